"""The 4-bit key/value cache's operators, as a program on this framework calls
them: rows appended to the cache, attention over it for single tokens and for
prompts (scores capped, biased by distance, masked by documents or a prefix),
the weights that each cached key has drawn, and the eviction that goes by them.

A case is one such call (an operator with the read-back of what it wrote, where
that is held in 4 bits).  Shapes are those of the repository's models (Qwen2-0.5B
14 query and 2 kv heads of width 64, GPT-2 124M 12 heads of width 64, the tiny
GPT-2 4 heads of width 32) and a generic grouped layer of 32 and 8 heads of width
128; positions run from none cached to 32768.  Keys get a spread of channel
magnitudes, as rotated keys have.

The cache's planes, for `capacity` positions (a multiple of 8) of each sequence
and kv head; blocks are 32 channels, a value is scale * (level - 8):
  k    [position][word g of 4][block][4 bytes]: channel 32 block + 8 g + i in nibble i
  v    [position / 8][n][pair of blocks][position % 8][2 bytes], n < min(16, width / 4):
       byte h, nibble e: channel 4 n_max pair + 2 n_max h + 2 n + e
  *_d  [position / 8][block][position % 8], f16
"""
import math
import os
import sys

import torch

own = False

MODELS = {"qwen2": (14, 2, 64), "gpt2": (12, 12, 64), "tiny": (4, 4, 32), "grouped": (32, 8, 128)}
ROPE_BASE = 10000.0


def listed():
    return [
        # one new token for each of 64 Qwen2 sequences: rotate, quantise, append
        {"name": "append_token", "kind": "append", "model": "qwen2", "seqs": 64, "rows": 1, "len": 511, "ragged": False,
         "tracked": True},
        # eight prompts of up to 1000 ids into empty caches
        {"name": "append_prompt", "kind": "append", "model": "grouped", "seqs": 8, "rows": 1000, "len": 0,
         "ragged": True, "tracked": False},
        # one sequence's decode step, the smallest attention
        {"name": "decode_one", "kind": "attention", "model": "qwen2", "seqs": 1, "rows": 1, "len": 511, "ragged": False,
         "cap": 0.0, "alibi": False, "mask": "causal"},
        # 64 sequences of different ages, the batched decode step
        {"name": "decode_batch", "kind": "attention", "model": "qwen2", "seqs": 64, "rows": 1, "len": 1023,
         "ragged": True, "cap": 0.0, "alibi": False, "mask": "causal"},
        # eight long contexts
        {"name": "decode_long", "kind": "attention", "model": "grouped", "seqs": 8, "rows": 1, "len": 32767,
         "ragged": True, "cap": 0.0, "alibi": False, "mask": "causal"},
        # one query head per kv head, capped scores, a distance bias and a sliding window
        {"name": "decode_capped", "kind": "attention", "model": "gpt2", "seqs": 16, "rows": 1, "len": 2999,
         "ragged": True, "cap": 30.0, "alibi": True, "mask": "window"},
        # packed documents with capped scores and padding rows that see nothing: the largest call
        {"name": "prompt_documents", "kind": "attention", "model": "grouped", "seqs": 4, "rows": 2048, "len": 0,
         "ragged": False, "cap": 50.0, "alibi": False, "mask": "documents"},
        # a later chunk of a prompt whose first rows see each other both ways
        {"name": "prompt_prefix", "kind": "attention", "model": "gpt2", "seqs": 2, "rows": 511, "len": 2000,
         "ragged": True, "cap": 0.0, "alibi": True, "mask": "prefix"},
        # a decode step that also keeps account of each key's weight
        {"name": "weigh_batch", "kind": "weigh", "model": "qwen2", "seqs": 64, "rows": 1, "len": 1023, "ragged": True,
         "cap": 0.0, "alibi": False, "mask": "causal"},
        # and a prompt's
        {"name": "weigh_prompt", "kind": "weigh", "model": "grouped", "seqs": 1, "rows": 1000, "len": 0,
         "ragged": False, "cap": 0.0, "alibi": False, "mask": "causal"},
        # eight long caches halved
        {"name": "evict_long", "kind": "evict", "model": "grouped", "seqs": 8, "rows": 1, "len": 16384, "ragged": True,
         "keep": 8192, "recent": 256},
        # 64 shorter ones of different lengths cut to 600 keys
        {"name": "evict_batch", "kind": "evict", "model": "qwen2", "seqs": 64, "rows": 1, "len": 1023, "ragged": True,
         "keep": 600, "recent": 64},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "weigh", "evict"])
    model = rng.choice(["qwen2", "qwen2", "grouped", "gpt2", "tiny"])
    n_heads, n_kv, hd = MODELS[model]
    room = 8 * 8 * 32768 * 128 // (n_kv * hd)  # cached positions over all sequences of the largest decode
    if kind == "append":
        rows = 1 if rng.random() < 0.5 else _log(rng, 2, 1000)
        return {"kind": kind, "model": model, "seqs": _log(rng, 1, 64 if rows == 1 else max(1, min(64, 8000 // rows))),
                "rows": rows, "len": rng.choice([0, 1, _log(rng, 2, 2000)]), "ragged": rng.random() < 0.5,
                "tracked": rng.random() < 0.5}
    if kind == "evict":
        length = _log(rng, 64, 16384)
        keep = max(1, int(length * rng.uniform(0.2, 0.9)))
        return {"kind": kind, "model": model, "seqs": _log(rng, 1, max(1, min(64, room // 4 // length))), "rows": 1,
                "len": length, "ragged": rng.random() < 0.7, "keep": keep, "recent": int(keep * rng.uniform(0.0, 0.6))}
    if kind == "decode" or (kind == "weigh" and rng.random() < 0.5):
        length = _log(rng, 1, 32767)
        seqs = _log(rng, 1, max(1, min(64, room // (length + 1))))
        rows = rng.choice([1, 1, 1, 2, 4])
    else:
        rows = _log(rng, 5, 2048)
        length = 0 if rng.random() < 0.6 else _log(rng, 1, 2000)
        most = 4 * 2048 * 2048 * 32 // 2
        seqs = _log(rng, 1, max(1, min(16, most // (rows * (rows + 2 * length) // 2 * n_heads + 1))))
    return {"kind": "weigh" if kind == "weigh" else "attention", "model": model, "seqs": seqs, "rows": rows,
            "len": length, "ragged": rng.random() < 0.5, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]),
            "alibi": rng.random() < 0.3,
            "mask": rng.choice(["causal", "causal", "window", "documents", "prefix"] if rows > 4 else
                               ["causal", "causal", "window"])}


# ---- what a case's sizes alone say ------------------------------------------


def _sizes(case):
    """Rows in use before the call and new rows of each sequence; the capacity."""
    n, rows, length = case["seqs"], case["rows"], case["len"]
    if not case["ragged"]:
        return [length] * n, [rows] * n, -(-(length + rows) // 8) * 8
    lens = [length - (length // 2) * i // max(1, n) - (i * i) % 5 * (length > 40) for i in range(n)]
    news = [rows - (rows // 2) * ((i * 5 + 1) % n) // n if rows > 4 else rows for i in range(n)]
    return lens, news, -(-(length + rows) // 8) * 8 + 8


def _allowed(case):
    """First and past-the-last cache row that each new row may see, per sequence."""
    lens, news, _ = _sizes(case)
    out = []
    for at, new in zip(lens, news):
        first, end = [0] * new, [at + t + 1 for t in range(new)]
        if case["mask"] == "window":
            wide = max(1, (at + new) // 2)
            first = [max(0, e - wide) for e in end]
        elif case["mask"] == "documents":
            part, t, j = max(3, new // 3), 0, 0
            while t < new:
                for u in range(t, min(new, t + part - j * 7 % 5)):
                    first[u] = at + t
                t, j = t + part - j * 7 % 5, j + 1
            for t in range(new - new // 50, new):  # padding at the end
                first[t] = end[t]
        elif case["mask"] == "prefix":
            end = [max(e, at + max(1, new // 4)) for e in end]
        out.append((first, end))
    return out


def work(case):
    n_heads, n_kv, hd = MODELS[case["model"]]
    lens, news, _ = _sizes(case)
    row = n_kv * hd * 2 * 0.5625  # bytes of one position's keys and values
    total = sum(news)
    if case["kind"] == "append":
        wide = (2 * n_heads + 2 * n_kv) * hd * 4 + row + (8 * n_kv if case["tracked"] else 0)
        back = case["seqs"] * case["rows"] * (row + 2 * n_kv * hd * 4)
        return {"bytes": total * wide + back, "flops": 6.0 * total * (n_heads + n_kv) * hd}
    if case["kind"] == "evict":
        kept = sum(min(x, case["keep"]) for x in lens)
        planes = kept * (2 * row + 16 * n_kv) + sum(lens) * n_kv * 4
        return {"bytes": planes + kept * (row + 2 * n_kv * hd * 4), "flops": 1.0 * sum(lens) * n_kv}
    pairs = seen = 0
    for first, end in _allowed(case):
        pairs += sum(max(0, e - f) for f, e in zip(first, end))
        seen += max(end) - min(first)
    by = seen * row + 2 * total * n_heads * hd * 4
    flops = 4.0 * hd * n_heads * pairs
    if case["kind"] == "weigh":
        by, flops = by + seen * n_kv * 8 + total * n_heads * 4, flops + 2.0 * hd * n_heads * pairs
    return {"bytes": by, "flops": flops}


# ---- the cache's format ------------------------------------------------------


def _levels(x):
    """Scales (f16) and levels 0 .. 15 of blocks of 32 channels: the scale is the
    first channel of largest magnitude over -8, the level the nearest one (the
    quotient in 64 bits, where no tie can be mistaken)."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(dim=-1, keepdim=True)
    at = (b.abs() == top).to(torch.uint8).argmax(dim=-1, keepdim=True)
    d = (b.gather(-1, at) / -8.0).to(torch.float16)
    w = d.double()
    q = torch.where(w != 0, torch.round(b.double() / torch.where(w != 0, w, 1.0)), 0.0).clamp(-8, 7) + 8
    return d.squeeze(-1), q.to(torch.uint8).reshape(x.shape)


def _planes(d_k, q_k, d_v, q_v):
    """The four planes of [seqs, kv heads, capacity, width] levels and their scales."""
    s, g, c, hd = q_k.shape
    nb, n = hd // 32, min(16, hd // 4)
    k = q_k.reshape(s, g, c, nb, 4, 4, 2).transpose(3, 4)
    v = q_v.reshape(s, g, c // 8, 8, hd // (4 * n), 2, n, 2).permute(0, 1, 2, 6, 4, 3, 5, 7)
    scales = lambda d: d.reshape(s, g, c // 8, 8, nb).transpose(3, 4).contiguous()  # noqa: E731
    nibbles = lambda x: (x[..., 0] | x[..., 1] << 4).contiguous().view(s, g, -1)  # noqa: E731
    return nibbles(k), scales(d_k), nibbles(v), scales(d_v)


def _unpack(plane):
    return torch.stack([plane & 15, plane >> 4], dim=-1).to(torch.float32) - 8.0


def _values(cache, upto):
    """Keys and values of the first `upto` positions (a multiple of 8) as f32, [seqs, kv heads, upto, width]."""
    s, g, hd = cache["k"].shape[0], cache["k"].shape[1], cache["hd"]
    nb, n = hd // 32, min(16, hd // 4)
    scale = lambda d: d[:, :, :upto // 8].to(torch.float32).transpose(3, 4).reshape(s, g, upto, nb, 1)  # noqa: E731
    k = _unpack(cache["k"][:, :, :upto * hd // 2]).reshape(s, g, upto, 4, nb, 8).transpose(3, 4)
    v = _unpack(cache["v"][:, :, :upto * hd // 2]).reshape(s, g, upto // 8, n, hd // (4 * n), 8, 2, 2)
    v = v.permute(0, 1, 2, 5, 4, 6, 3, 7)
    k = k.reshape(s, g, upto, nb, 32) * scale(cache["k_d"])
    v = v.reshape(s, g, upto, nb, 32) * scale(cache["v_d"])
    return k.reshape(s, g, upto, hd), v.reshape(s, g, upto, hd)


# ---- inputs ------------------------------------------------------------------


def _filled(gen, seqs, n_kv, cap, hd):
    """A cache whose every position holds quantised keys and values."""
    parts = []
    spread = torch.exp(0.4 * torch.randn((n_kv, 1, hd), generator=gen, device="cuda"))
    for _ in range(seqs):
        k = torch.randn((1, n_kv, cap, hd), generator=gen, device="cuda") * spread
        v = torch.randn((1, n_kv, cap, hd), generator=gen, device="cuda")
        parts.append(_planes(*_levels(k), *_levels(v)))
    k, k_d, v, v_d = (torch.cat(p) for p in zip(*parts))
    return {"k": k, "k_d": k_d, "v": v, "v_d": v_d, "hd": hd, "pos": None, "weight": None}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n_heads, n_kv, hd = MODELS[case["model"]]
    lens, news, cap = _sizes(case)
    seqs, total = case["seqs"], sum(news)
    s = {"case": case, "cache": _filled(gen, seqs, n_kv, cap, hd), "len": _ints(lens), "cap": cap,
         "off": _ints([sum(news[:i]) for i in range(seqs + 1)]) if case["ragged"] else None, "total": total}
    tracked = case["kind"] in ("weigh", "evict") or case.get("tracked")
    if tracked:
        s["cache"]["pos"] = torch.arange(cap, dtype=torch.int32, device="cuda").expand(seqs, n_kv, cap).contiguous()
        s["cache"]["weight"] = torch.rand((seqs, n_kv, cap), generator=gen, device="cuda") ** 4
    # where each new row sits in a [seqs, rows] grid
    s["slot"] = torch.cat([torch.arange(n, device="cuda") + i * case["rows"] for i, n in enumerate(news)])
    s["at"] = _ints([a + t for a, n in zip(lens, news) for t in range(n)])  # each new row's position
    if case["kind"] == "append":
        s["qkv"] = torch.randn((total, (n_heads + 2 * n_kv) * hd), generator=gen, device="cuda")
        s["q"] = torch.empty((total, n_heads * hd), device="cuda")
        s["k_out"] = torch.empty((seqs, case["rows"], n_kv * hd), device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    elif case["kind"] == "evict":
        kcap = -(-case["keep"] // 8) * 8
        s["to"] = {"k": torch.zeros((seqs, n_kv, kcap * hd // 2), dtype=torch.uint8, device="cuda"), "hd": hd,
                   "k_d": torch.zeros((seqs, n_kv, kcap // 8, hd // 32, 8), dtype=torch.float16, device="cuda"),
                   "pos": torch.zeros((seqs, n_kv, kcap), dtype=torch.int32, device="cuda"),
                   "weight": torch.zeros((seqs, n_kv, kcap), device="cuda")}
        s["to"]["v"], s["to"]["v_d"] = torch.zeros_like(s["to"]["k"]), torch.zeros_like(s["to"]["k_d"])
        s["new_len"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        s["k_out"] = torch.empty((seqs, case["keep"], n_kv * hd), device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        s["q"] = torch.randn((total, n_heads * hd), generator=gen, device="cuda")
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((total, n_heads), device="cuda") if case["kind"] == "weigh" else None
        bounds = _allowed(case)
        masked = case["mask"] != "causal"
        s["first"] = _ints([x for f, _ in bounds for x in f]) if masked else None
        s["end"] = _ints([x for _, e in bounds for x in e]) if masked else None
        s["slopes"] = None
        if case["alibi"]:
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, n_heads + 1, device="cuda") / n_heads)
    return s


# ---- the plain forms ---------------------------------------------------------


def _rotated(x, at, hd):
    """Split-half rotation of [rows, heads, hd]; the angle is the framework's (position and
    frequency in 32 bits), the rest in 64 bits: a key's channels go on to a level's border."""
    half = hd // 2
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    freq = torch.pow(torch.full_like(i, ROPE_BASE), -2.0 * i / hd).to(torch.float32)
    angle = (at.to(torch.float32)[:, None] * freq).double()[:, None]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], dim=-1).float()


def _plain_append(s):
    case = s["case"]
    n_heads, n_kv, hd = MODELS[case["model"]]
    seqs, rows, cap, c = case["seqs"], case["rows"], s["cap"], s["cache"]
    nb, n = hd // 32, min(16, hd // 4)
    q, k, v = s["qkv"].view(s["total"], -1, hd).split([n_heads, n_kv, n_kv], dim=1)
    seq, at = s["slot"] // rows, s["at"].long()
    q, k = _rotated(q, at, hd), _rotated(k, at, hd)
    (d_k, q_k), (d_v, q_v) = _levels(k), _levels(v)
    nibbles = lambda x: x[..., 0] | x[..., 1] << 4  # noqa: E731
    k_bytes = nibbles(q_k.reshape(-1, n_kv, nb, 4, 4, 2).transpose(2, 3)).reshape(-1, n_kv, hd // 2)
    v_bytes = nibbles(q_v.reshape(-1, n_kv, hd // (4 * n), 2, n, 2).permute(0, 1, 4, 2, 3, 5))
    c["k"].view(seqs, n_kv, cap, hd // 2)[seq, :, at] = k_bytes
    c["v"].view(seqs, n_kv, cap // 8, hd // 4, 8, 2)[seq, :, at // 8, :, at % 8] = v_bytes.reshape(-1, n_kv, hd // 4, 2)
    c["k_d"][seq, :, at // 8, :, at % 8] = d_k
    c["v_d"][seq, :, at // 8, :, at % 8] = d_v
    if c["pos"] is not None:
        c["pos"][seq, :, at] = s["at"][:, None].expand(-1, n_kv)
        c["weight"][seq, :, at] = 0.0
    out = {"q": q.reshape(s["total"], -1), "pos": c["pos"], "weight": c["weight"]}
    # (positions past the capacity, which a shorter sequence's grid reaches, read as NaN)
    where = s["len"].long()[:, None] + torch.arange(rows, device="cuda")
    ok = (where < cap)[:, None, :, None]
    where = where.clamp(max=cap - 1)[:, None, :, None].expand(-1, n_kv, -1, hd)
    for name, x in zip(("k_out", "v_out"), _values(c, cap)):
        x = torch.where(ok, x.gather(2, where), math.nan)
        out[name] = x.transpose(1, 2).reshape(seqs, rows, n_kv * hd)
    return out


def _plain_attention(s):
    case = s["case"]
    n_heads, n_kv, hd = MODELS[case["model"]]
    seqs, rows, group = case["seqs"], case["rows"], n_heads // n_kv
    upto = -(-(case["len"] + rows) // 8) * 8
    k, v = _values(s["cache"], upto)

    def grid(x, fill):  # [rows in use, ...] in the [seqs, rows] grid
        y = torch.full((seqs * rows, *x.shape[1:]), fill, dtype=x.dtype, device="cuda")
        y[s["slot"]] = x
        return y.view(seqs, rows, *x.shape[1:])

    q = grid(s["q"], 0.0).view(seqs, rows, n_kv, group, hd).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.reshape(seqs, n_kv, group * rows, hd), k.transpose(2, 3)) / math.sqrt(hd)
    scores = scores.view(seqs, n_kv, group, rows, upto)
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    here = torch.arange(upto, device="cuda")
    at = grid(s["at"].long(), 0)
    if s["slopes"] is not None:
        far = (at[:, :, None] - here).abs().to(torch.float32)
        scores = scores - s["slopes"].view(1, n_kv, group, 1, 1) * far[:, None, None]
    first = grid(s["first"].long(), 0) if s["first"] is not None else torch.zeros_like(at)
    end = grid(s["end"].long(), 0) if s["end"] is not None else at + 1
    seen = ((here >= first[:, :, None]) & (here < end[:, :, None]))[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(scores - top)
    mass = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(mass > 0, mass, 1.0)
    o = torch.matmul(p.view(seqs, n_kv, group * rows, upto), v).view(seqs, n_kv, group, rows, hd)
    out = {"out": o.permute(0, 3, 1, 2, 4).reshape(seqs * rows, n_heads * hd)[s["slot"]]}
    if case["kind"] == "weigh":
        lse = (top + torch.log(mass)).squeeze(-1)  # (log 0: a row that sees nothing)
        out["lse"] = lse.permute(0, 3, 1, 2).reshape(seqs * rows, n_heads)[s["slot"]]
        real = grid(torch.ones_like(s["at"], dtype=torch.bool), False)
        p = torch.where(real[:, None, None, :, None], p, 0.0)
        s["cache"]["weight"][:, :, :upto] += p.sum(dim=(2, 3))
        out["weight"] = s["cache"]["weight"]
    return out


def _by_position(plane, positions, octets):
    """A plane as [seqs, kv heads, positions, values]: a view, or where eight positions lie side by side a copy."""
    if not octets:
        return plane.view(*plane.shape[:2], positions, -1)
    return plane.reshape(*plane.shape[:2], positions // 8, -1, 8, octets).transpose(3, 4).flatten(4).flatten(2, 3)


def _plain_evict(s):
    case, c, to = s["case"], s["cache"], s["to"]
    n_kv, hd, cap, kcap = c["k"].shape[1], c["hd"], s["cap"], s["to"]["pos"].shape[2]
    seqs, keep = case["seqs"], case["keep"]
    length = s["len"].long()[:, None, None]
    here = torch.arange(cap, device="cuda")
    rank = torch.where(here >= length - case["recent"], math.inf, c["weight"])
    rank = torch.where(here < length, rank, -math.inf)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values
    kept = torch.where(length <= keep, here[:keep], kept)
    ok = (here[:keep] < length).expand(-1, n_kv, -1)[..., None]  # (rows past a short cache's end stay as they were)

    def moved(name, octets=0):
        src, old = _by_position(c[name], cap, octets), _by_position(to[name], kcap, octets)[:, :, :keep]
        return torch.where(ok, src.gather(2, kept[..., None].expand(-1, -1, -1, src.shape[3])), old)

    at = torch.arange(keep, device="cuda")
    for name in ("k", "pos", "weight"):
        to[name].view(seqs, n_kv, kcap, -1)[:, :, :keep] = moved(name)
    for name, octets in (("v", 2), ("k_d", 1), ("v_d", 1)):
        plane = to[name].view(seqs, n_kv, kcap // 8, -1, 8, octets)
        plane[:, :, at // 8, :, at % 8] = moved(name, octets).view(seqs, n_kv, keep, -1, octets).permute(2, 0, 1, 3, 4)
    s["new_len"].copy_(s["len"].clamp(max=keep))
    k, v = (x[:, :, :keep].transpose(1, 2).reshape(seqs, keep, n_kv * hd) for x in _values(to, kcap))
    return {"k_out": k, "v_out": v, "pos": to["pos"], "weight": to["weight"], "new_len": s["new_len"]}


# ---- one pass ----------------------------------------------------------------

_kept = []


def _framework():
    """The framework and the program's one context, on torch's stream."""
    if not _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "ferrum-cpu_amd"))
        import ferrum_hip as fh

        ctx = fh.Context(0)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        _kept.extend((fh, ctx))
    return _kept


def _handle(fh, c, n_kv, capacity):
    """The framework's view of a cache, made once."""
    if "handle" not in c:
        c["handle"] = fh.KV4Cache(c["k"].shape[0], n_kv, c["hd"], capacity, c["k"], c["k_d"], c["v"], c["v_d"], c["pos"],
                                  c["weight"])
    return c["handle"]


def _own(s):
    fh, ctx = _framework()
    case = s["case"]
    n_heads, n_kv, hd = MODELS[case["model"]]
    cache = _handle(fh, s["cache"], n_kv, s["cap"])
    rows, total = case["rows"], s["total"]
    if case["kind"] == "append":
        fh.kv4_append_async(ctx, cache, s["qkv"], (n_heads + 2 * n_kv) * hd, total, n_heads, s["off"], rows, s["len"],
                            s["at"], hd, ROPE_BASE, fh.ROPE_NEOX, None, 1.0, s["q"])
        fh.kv4_read_async(ctx, cache, s["len"], rows, s["k_out"], s["v_out"])
        return {"q": s["q"], "k_out": s["k_out"], "v_out": s["v_out"], "pos": s["cache"]["pos"],
                "weight": s["cache"]["weight"]}
    if case["kind"] == "evict":
        to = _handle(fh, s["to"], n_kv, s["to"]["pos"].shape[2])
        fh.kv4_evict_async(ctx, cache, to, s["len"], case["len"], case["keep"], case["recent"], s["new_len"])
        fh.kv4_read_async(ctx, to, None, case["keep"], s["k_out"], s["v_out"])
        return {"k_out": s["k_out"], "v_out": s["v_out"], "pos": s["to"]["pos"], "weight": s["to"]["weight"],
                "new_len": s["new_len"]}
    if "score" not in s:
        s["score"] = fh.AttnScore(case["cap"], s["slopes"], None, s["first"], s["end"])
    fh.kv4_attention_async(ctx, cache, s["q"], n_heads * hd, total, n_heads, s["off"], rows, s["len"],
                           case["len"] + rows, s["score"], s["out"], s["lse"])
    if case["kind"] == "attention":
        return {"out": s["out"]}
    fh.kv4_weigh_async(ctx, cache, s["q"], n_heads * hd, total, n_heads, s["off"], rows, s["len"], case["len"] + rows,
                       s["score"], s["lse"])
    return {"out": s["out"], "lse": s["lse"], "weight": s["cache"]["weight"]}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    return _plain_append(state) if kind == "append" else _plain_evict(state) if kind == "evict" else _plain_attention(state)


# ---- from the definitions, in 64 bits ----------------------------------------


def _exact_plane(plane, d, i, hd, keys, v):
    """Positions `keys` of sequence i's plane as float64, [kv heads, keys, hd], by each channel's place."""
    c = torch.arange(hd, device="cuda")
    key = keys[:, None]
    if v:
        n_max = min(16, hd // 4)
        pair, half = c // (4 * n_max), c % (4 * n_max) // (2 * n_max)
        n, e = c % (2 * n_max) // 2, c % 2
        where = (((key // 8) * n_max + n) * (hd // (4 * n_max)) + pair) * 16 + key % 8 * 2 + half
        shift = 4 * e
    else:
        where = key * (hd // 2) + (c % 32 // 8 * (hd // 32) + c // 32) * 4 + c % 8 // 2
        shift = c % 2 * 4
    level = plane[i][:, where] >> shift & 15
    scale = d[i].flatten(1)[:, (key // 8 * (hd // 32) + c // 32) * 8 + key % 8]
    return (level.double() - 8) * scale.double()


def _exact_levels(x):
    """What x's blocks stand for once quantised, in float64."""
    b = x.unflatten(-1, (-1, 32))
    most, _ = b.abs().max(dim=-1, keepdim=True)
    first = (b.abs() >= most).long().cumsum(-1).eq(0).sum(-1, keepdim=True)
    d = torch.take_along_dim(b, first, -1).div(-8).half().double()
    level = torch.where(d == 0, torch.zeros_like(b, dtype=torch.float64), (b.double() / d).round().clamp(-8, 7))
    return (level * d).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    n_heads, n_kv, hd = MODELS[case["model"]]
    lens, news, cap = _sizes(case)
    c, group = s["cache"], n_heads // n_kv
    if case["kind"] == "append":
        x = s["qkv"].view(s["total"], n_heads + 2 * n_kv, hd)
        ks, vs, row = [], [], 0
        p = torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd
        freq = torch.tensor(ROPE_BASE, dtype=torch.float64, device="cuda").pow(-p).float()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           (s["at"].float()[:, None] * freq).double())[:, None]
        z = torch.complex(*x[:, :n_heads + n_kv].double().chunk(2, dim=-1)) * turn
        z = torch.cat([z.real, z.imag], dim=-1)
        for i, (at, new) in enumerate(zip(lens, news)):
            keys = at + torch.arange(case["rows"], device="cuda")
            kv = []
            for name, y in (("k", z[row:row + new, n_heads:].float()), ("v", x[row:row + new, n_heads + n_kv:])):
                old = _exact_plane(c[name], c[name + "_d"], i, hd, keys.clamp(max=cap - 1), name == "v")
                old[:, keys >= cap] = math.nan
                old[:, :new] = _exact_levels(y).transpose(0, 1)
                kv.append(old.transpose(0, 1).flatten(1))
            ks.append(kv[0])
            vs.append(kv[1])
            row += new
        out = {"q": z[:, :n_heads].flatten(1), "k_out": torch.stack(ks), "v_out": torch.stack(vs), "pos": None}
        if c["pos"] is not None:
            w, row = c["weight"].double(), 0
            for i, (at, new) in enumerate(zip(lens, news)):
                w[i, :, at:at + new] = 0
            out["weight"] = w
        return out
    if case["kind"] == "evict":
        keep, kcap = case["keep"], s["to"]["pos"].shape[2]
        k = torch.zeros((case["seqs"], keep, n_kv, hd), dtype=torch.float64, device="cuda")
        v, w = torch.zeros_like(k), torch.zeros((case["seqs"], n_kv, kcap), dtype=torch.float64, device="cuda")
        for i, at in enumerate(lens):
            weight = c["weight"][i, :, :at].cpu().numpy()
            for h in range(n_kv):
                kept = list(range(at))
                if at > keep:
                    free = at - case["recent"]
                    heavy = sorted(range(free), key=lambda j: (-weight[h, j], j))[:keep - case["recent"]]
                    kept = sorted(heavy) + list(range(free, at))
                kept = torch.tensor(kept, device="cuda")
                one = lambda n: _exact_plane(c[n][:, h:h + 1], c[n + "_d"][:, h:h + 1], i, hd, kept, n == "v")[0]  # noqa
                k[i, :len(kept), h], v[i, :len(kept), h] = one("k"), one("v")
                w[i, h, :len(kept)] = c["weight"][i, h, kept].double()
        return {"k_out": k.flatten(2), "v_out": v.flatten(2), "pos": None, "weight": w, "new_len": None}
    outs, lses, row = [], [], 0
    weights = c["weight"].double() if c["weight"] is not None else None
    for i, ((first, end), at, new) in enumerate(zip(_allowed(case), lens, news)):
        upto = max(end)
        keys = torch.arange(upto, device="cuda")
        k, v = (_exact_plane(c[n], c[n + "_d"], i, hd, keys, n == "v") for n in ("k", "v"))
        lo, hi = (torch.tensor(x, device="cuda")[:, None] for x in (first, end))
        me = at + torch.arange(new, device="cuda")[:, None]
        hidden = (keys < lo) | (keys >= hi)
        x = s["q"][row:row + new].double().view(new, n_heads, hd)
        heads, tops = [], []
        for h in range(n_heads):
            z = x[:, h] @ k[h // group].T * hd ** -0.5
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if case["alibi"]:
                z -= (me - keys).abs() * s["slopes"][h].double()
            z.masked_fill_(hidden, -math.inf)
            lse = torch.logsumexp(z, dim=1, keepdim=True)
            p = torch.where(hidden, 0.0, torch.exp(z - lse))
            heads.append(p @ v[h // group])
            tops.append(lse)
            if weights is not None:
                weights[i, h // group, :upto] += p.sum(0)
        outs.append(torch.cat(heads, dim=1))
        lses.append(torch.cat(tops, dim=1))
        row += new
    out = {"out": torch.cat(outs)}
    if case["kind"] == "weigh":
        out.update(lse=torch.cat(lses), weight=weights)
    return out
