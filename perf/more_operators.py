"""Serving a Llama-shaped model from its f32 key/value cache with drafted tokens, as
a program on this framework calls it: prompts of different lengths at once, a tree
of drafted tokens over each sequence's cache, the acceptance of what the model
agreed with (its rows moved together in every layer's cache), and the edits that
logits get before they are sampled (penalties, biases, grammar masks).

A case is one such call.  Shapes are those of the repository's models (Qwen2-0.5B 14
query and 2 kv heads of width 64, GPT-2 124M 12 heads of width 64, the tiny GPT-2 4
heads of width 32) and a generic grouped layer of 32 and 8 heads of width 128;
vocabularies are GPT-2's and Qwen2's.
"""
import math
import os
import random
import sys

import torch

own = False

# query heads, kv heads, width, rotation: split halves, neighbours, or none
MODELS = {"qwen2": (14, 2, 64, "neox"), "gpt2": (12, 12, 64, None), "tiny": (4, 4, 32, "neox"),
          "grouped": (32, 8, 128, "norm")}
ROPE_BASE = 10000.0


def listed():
    return [
        # a short question to an idle server: the smallest prompt
        {"name": "prompt_one", "kind": "prompt", "model": "qwen2", "seqs": 1, "rows": 64, "len": 0, "ragged": False},
        # sixteen prompts of different lengths fed together
        {"name": "prompt_packed", "kind": "prompt", "model": "qwen2", "seqs": 16, "rows": 1000, "len": 0, "ragged": True},
        # a later chunk of two long prompts, one query head to a kv head
        {"name": "prompt_chunk", "kind": "prompt", "model": "gpt2", "seqs": 2, "rows": 511, "len": 2000, "ragged": True},
        # one long document: the largest call
        {"name": "prompt_long", "kind": "prompt", "model": "grouped", "seqs": 1, "rows": 8192, "len": 0, "ragged": False},
        # one sequence's drafted tree
        {"name": "tree_one", "kind": "tree", "model": "qwen2", "seqs": 1, "rows": 16, "len": 511, "ragged": False},
        # trees of different sizes over 32 sequences of different ages
        {"name": "tree_batch", "kind": "tree", "model": "qwen2", "seqs": 32, "rows": 32, "len": 1023, "ragged": True},
        # large trees over four long contexts
        {"name": "tree_long", "kind": "tree", "model": "grouped", "seqs": 4, "rows": 64, "len": 16383, "ragged": True},
        # what one sequence accepted, in the caches of 24 layers
        {"name": "accept_one", "kind": "accept", "model": "qwen2", "seqs": 1, "rows": 16, "len": 511, "ragged": False,
         "layers": 24},
        # and 32 sequences
        {"name": "accept_batch", "kind": "accept", "model": "qwen2", "seqs": 32, "rows": 32, "len": 255, "ragged": True,
         "layers": 24},
        # one chat turn's penalties and a few biased tokens
        {"name": "edit_one", "kind": "edit", "vocab": 50257, "seqs": 1, "rows": 1, "history": 300, "biases": 16,
         "masks": 0},
        # a batched step: long histories, biases, and half the rows under a grammar
        {"name": "edit_batch", "kind": "edit", "vocab": 151936, "seqs": 64, "rows": 1, "history": 1000, "biases": 100,
         "masks": 32},
        # the nodes of eight drafted trees, each with its own path and its own grammar state
        {"name": "edit_tree", "kind": "edit", "vocab": 151936, "seqs": 8, "rows": 32, "history": 500, "biases": 0,
         "masks": 256},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "tree", "tree", "accept", "edit", "edit"])
    if kind == "edit":
        rows = rng.choice([1, 1, _log(rng, 2, 64)])
        vocab = rng.choice([50257, 151936, _log(rng, 100, 151936)])
        seqs = _log(rng, 1, max(1, min(64, 256 // rows)))
        return {"kind": kind, "vocab": vocab, "seqs": seqs, "rows": rows, "history": rng.choice([0, _log(rng, 1, 4000)]),
                "biases": rng.choice([0, _log(rng, 1, min(300, vocab))]),
                "masks": rng.choice([0, 1, seqs * rows, max(1, seqs * rows // 2)])}
    model = rng.choice(["qwen2", "qwen2", "grouped", "gpt2", "tiny"])
    n_heads, n_kv, hd, _ = MODELS[model]
    case = {"kind": kind, "model": model, "ragged": rng.random() < 0.6}
    if kind == "prompt":
        case["rows"] = _log(rng, 1, 8192)
        case["len"] = 0 if rng.random() < 0.6 else _log(rng, 1, 4000)
        most = 8192 * 8192 // 2 * 32 * 128 // 2
        pairs = case["rows"] * (case["rows"] + 2 * case["len"]) // 2 * n_heads * hd
        case["seqs"] = _log(rng, 1, max(1, min(32, most // (pairs + 1), 32768 // (case["rows"] + case["len"]))))
        return case
    case["rows"] = _log(rng, 1, 64)
    if kind == "tree":
        case["len"] = _log(rng, 1, 16383)
        case["seqs"] = _log(rng, 1, max(1, min(64, 4 * 16384 * 1024 // ((case["len"] + case["rows"]) * n_kv * hd))))
        return case
    case["len"], case["layers"] = _log(rng, 1, 1000), rng.choice([2, 12, 24])
    room = 32 * 288 * 128 * 24
    case["seqs"] = _log(rng, 1, max(1, min(64, room // ((case["len"] + case["rows"]) * n_kv * hd * case["layers"]))))
    return case


# ---- what a case's sizes alone say ------------------------------------------


def _sizes(case):
    """Rows in use before the call and new rows of each sequence; the capacity."""
    n, rows, length = case["seqs"], case["rows"], case["len"]
    if not case["ragged"]:
        return [length] * n, [rows] * n, length + rows
    lens = [length - (length // 2) * i // n - (i * i) % 5 * (length > 40) for i in range(n)]
    news = [rows - (rows // 2) * ((i * 5 + 1) % n) // n for i in range(n)]
    return lens, news, length + rows + 5


def _parents(n, i):
    """A drafted tree of n nodes: each node's parent is one of the eight before it."""
    rng = random.Random(1000 * n + i)
    return [-1] + [rng.randrange(max(0, t - 8), t) for t in range(1, n)]


def _path(parents, t):
    out = [t]
    while parents[t] >= 0:
        t = parents[t]
        out.append(t)
    return out[::-1]


def _accepted(n, i):
    """The path that sequence i's tree will be accepted along: at most eight nodes,
    none of which lies where another is moved to, so that a pass can be repeated."""
    parents = _parents(n, i)
    paths = [_path(parents, t) for t in range(n)]
    paths = [p for p in paths if len(p) <= 8 and all(x == j or x >= len(p) for j, x in enumerate(p))]
    return random.Random(77 * n + i).choice(paths)


def work(case):
    if case["kind"] == "edit":
        rows, v = case["seqs"] * case["rows"], case["vocab"]
        lists = case["seqs"] * case["history"] * 4 + rows * (case["biases"] * 8 + 28)
        return {"bytes": rows * v * 8 + case["masks"] * (-(-v // 32)) * 4 + lists, "flops": 4.0 * rows * v}
    n_heads, n_kv, hd, _ = MODELS[case["model"]]
    lens, news, _ = _sizes(case)
    if case["kind"] == "accept":
        moved = sum(sum(x != j for j, x in enumerate(_accepted(n, i))) for i, n in enumerate(news))
        return {"bytes": sum(news) * 16 + case["seqs"] * 16 + moved * case["layers"] * 2 * n_kv * hd * 8, "flops": 0.0}
    total = sum(news)
    if case["kind"] == "tree":
        pairs = sum(n * at + sum(len(_path(_parents(n, i), t)) for t in range(n)) for i, (at, n) in enumerate(zip(lens, news)))
    else:
        pairs = sum(n * at + n * (n + 1) // 2 for at, n in zip(lens, news))
    # q|k|v in, the outputs and the new cache rows out, the cached rows in
    bytes_ = total * (2 * n_heads + 4 * n_kv) * hd * 4 + sum(lens) * 2 * n_kv * hd * 4
    return {"bytes": bytes_, "flops": 4.0 * hd * n_heads * pairs}


# ---- inputs ------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_edit(case, gen):
    seqs, n, v = case["seqs"], case["rows"], case["vocab"]
    rows = seqs * n
    rand = lambda *shape: torch.rand(shape, generator=gen, device="cuda")  # noqa: E731
    ids = lambda *shape: torch.randint(0, v, shape, generator=gen, device="cuda", dtype=torch.int32)  # noqa: E731
    s = {"case": case, "logits": 3.0 * torch.randn((rows, v), generator=gen, device="cuda")}
    s["out"] = torch.empty_like(s["logits"])
    # histories of text: a few ids come often
    s["recent"] = (rand(seqs, max(1, case["history"])) ** 3 * v).to(torch.int32).clamp(max=v - 1)
    lens = [case["history"] - case["history"] * (i % 4) // 8 for i in range(seqs)]
    first = [i * max(1, case["history"]) for i in range(seqs)]
    s["ranges"] = _ints([[first[r // n], first[r // n] + lens[r // n]] for r in range(rows)])
    s["repetition"], s["frequency"], s["presence"] = 1.0 + 0.3 * rand(rows), 0.5 * rand(rows), 0.5 * rand(rows)
    if n > 1:
        s["parent"] = _ints([p for i in range(seqs) for p in _parents(n, i)])
        s["tokens"] = ids(rows)
    if case["biases"]:
        s["bias_off"] = _ints([r * case["biases"] for r in range(rows + 1)])
        start = torch.randint(0, v, (rows, 1), generator=gen, device="cuda")
        step = max(1, v // case["biases"])  # distinct ids of a row
        s["bias_id"] = ((start + step * torch.arange(case["biases"], device="cuda")) % v).to(torch.int32).flatten()
        s["bias"] = 4.0 * torch.randn(rows * case["biases"], generator=gen, device="cuda")
    if case["masks"]:
        # a grammar's state allows a few ids or nearly all of them
        allow = rand(case["masks"], -(-v // 32), 32) < torch.where(rand(case["masks"], 1, 1) < 0.5, 0.02, 0.9)
        bits = torch.bitwise_left_shift(allow.to(torch.int64), torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = (bits - ((bits >> 31) << 32)).to(torch.int32)
        s["mask_of"] = _ints([r if r < case["masks"] else -1 for r in range(rows)])
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "edit":
        return _prepare_edit(case, gen)
    n_heads, n_kv, hd, _ = MODELS[case["model"]]
    lens, news, cap = _sizes(case)
    seqs, total = case["seqs"], sum(news)
    s = {"case": case, "len": _ints(lens), "cap": cap, "total": total,
         "off": _ints([sum(news[:i]) for i in range(seqs + 1)]) if case["ragged"] else None}
    if case["kind"] != "prompt":
        s["parent"] = _ints([p for i, n in enumerate(news) for p in _parents(n, i)])
    if case["kind"] == "accept":
        s["tokens"] = torch.randint(0, 151936, (total,), generator=gen, device="cuda", dtype=torch.int32)
        s["chosen"] = torch.randint(0, 151936, (total,), generator=gen, device="cuda", dtype=torch.int32)
        first, src, dst = 0, [], []
        for i, n in enumerate(news):
            p = _accepted(n, i)
            dst += [first + x for x in p[:-1]]
            src += [first + x for x in p[1:]]
            first += n
        s["chosen"][_ints(dst).long()] = s["tokens"][_ints(src).long()]
        planes = 2 * case["layers"]
        s["cache"] = torch.randn((planes, seqs, cap, n_kv * hd), generator=gen, device="cuda")
        s["planes"] = torch.tensor([s["cache"][p].data_ptr() for p in range(planes)], dtype=torch.int64, device="cuda")
        s["path"], s["count"] = torch.empty_like(s["tokens"]), torch.empty_like(s["len"])
        s["next"], s["new_len"] = torch.empty_like(s["len"]), torch.empty_like(s["len"])
        return s
    # keys get a spread of channel magnitudes, as rotated keys have
    spread = torch.exp(0.4 * torch.randn((n_kv * hd), generator=gen, device="cuda"))
    s["k"], s["v"] = (torch.zeros((seqs, cap, n_kv * hd), device="cuda") for _ in range(2))
    for i, at in enumerate(lens):
        s["k"][i, :at] = torch.randn((at, n_kv * hd), generator=gen, device="cuda") * spread
        s["v"][i, :at] = torch.randn((at, n_kv * hd), generator=gen, device="cuda")
    s["qkv"] = torch.randn((total, (n_heads + 2 * n_kv) * hd), generator=gen, device="cuda")
    s["qkv"][:, n_heads * hd:(n_heads + n_kv) * hd] *= spread
    s["out"] = torch.empty((total, n_heads * hd), device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------


def _rotated(x, at, hd, kind):
    """Rotation of [rows, heads, hd]; the angle is the framework's (position and frequency
    in 32 bits), its sine and cosine in 64 bits."""
    if kind is None:
        return x
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    freq = torch.pow(torch.full_like(i, ROPE_BASE), -2.0 * i / hd).to(torch.float32)
    angle = (at.to(torch.float32)[:, None] * freq).double()[:, None]
    c, sn = angle.cos().float(), angle.sin().float()
    if kind == "neox":
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat([a * c - b * sn, a * sn + b * c], dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * sn, a * sn + b * c], dim=-1).flatten(-2)


def _ancestors(parent):
    """[n, n]: whether a node's path holds another (itself among them)."""
    n = parent.shape[0]
    seen = torch.eye(n, dtype=torch.bool, device="cuda")
    up = parent.long()
    for t in range(1, n):
        seen[t] |= seen[up[t].clamp(min=0)] & (up[t] >= 0)
    return seen


def _plain_attention(s):
    case = s["case"]
    n_heads, n_kv, hd, rope = MODELS[case["model"]]
    lens, news, _ = _sizes(case)
    group, row = n_heads // n_kv, 0
    q, k, v = s["qkv"].view(s["total"], -1, hd).split([n_heads, n_kv, n_kv], dim=1)
    out = torch.empty((s["total"], n_heads, hd), device="cuda")
    for i, (at, new) in enumerate(zip(lens, news)):
        mine, upto = slice(row, row + new), at + new
        here = torch.arange(new, device="cuda")
        if case["kind"] == "tree":
            own_seen = _ancestors(s["parent"][mine])
            where = at + own_seen.sum(1) - 1
        else:
            own_seen = here[:, None] >= here
            where = at + here
        seen = torch.cat([torch.ones((new, at), dtype=torch.bool, device="cuda"), own_seen], dim=1)
        qr, kr = _rotated(q[mine], where, hd, rope), _rotated(k[mine], where, hd, rope)
        s["k"][i, at:upto] = kr.flatten(1)
        s["v"][i, at:upto] = v[mine].flatten(1)
        for g in range(n_kv):
            keys, values = (s[c][i, :upto, g * hd:(g + 1) * hd] for c in "kv")
            for h in range(g * group, (g + 1) * group):
                x = torch.matmul(qr[:, h], keys.T.contiguous()) / math.sqrt(hd)
                x = torch.where(seen, x, -math.inf)
                p = torch.exp(x - x.amax(dim=-1, keepdim=True))
                p = p / p.sum(dim=-1, keepdim=True)
                out[mine, h] = torch.matmul(p, values)
        row += new
    return {"out": out.flatten(1), "k": s["k"], "v": s["v"]}


def _plain_accept(s):
    case = s["case"]
    _, news, _ = _sizes(case)
    seqs, rows = case["seqs"], max(news)
    slot = torch.cat([torch.arange(n, device="cuda") + i * rows for i, n in enumerate(news)])

    def grid(x, fill):
        y = torch.full((seqs * rows,), fill, dtype=torch.int64, device="cuda")
        y[slot] = x.long()
        return y.view(seqs, rows)

    parent, tokens, chosen = grid(s["parent"], -1), grid(s["tokens"], -1), grid(s["chosen"], -2)
    up = parent.clamp(min=0)
    match = (tokens == chosen.gather(1, up)) & (parent >= 0)
    # the first matching child of each node
    t = torch.arange(rows, device="cuda")
    best = torch.full((seqs, rows), rows, dtype=torch.int64, device="cuda")
    best.scatter_reduce_(1, up, torch.where(match, t, rows), "amin")
    link = match & (best.gather(1, up) == t)
    taken = torch.zeros((seqs, rows), dtype=torch.bool, device="cuda")
    taken[:, 0] = True
    for j in range(1, rows):
        taken[:, j] = link[:, j] & taken.gather(1, up[:, j:j + 1])[:, 0]
    count = taken.sum(1)
    last = torch.where(taken, t, 0).amax(1)
    path = torch.where(taken, t, rows).sort(dim=1).values
    path = torch.where(path < rows, path, -1)
    base = s["len"].long()[:, None]
    cap = s["cap"]
    src = torch.where(path >= 0, base + path, base + t).clamp(max=cap - 1)
    seq = torch.arange(seqs, device="cuda")[:, None]
    moved = s["cache"][:, seq, src]
    ok = (path >= 0)[None, :, :, None]
    dst = (base + t).clamp(max=cap - 1)
    s["cache"][:, seq, dst] = torch.where(ok, moved, s["cache"][:, seq, dst])
    return {"path": path.flatten()[slot].to(torch.int32), "count": count.to(torch.int32),
            "next": chosen.gather(1, last[:, None])[:, 0].to(torch.int32),
            "new_len": (s["len"] + count).to(torch.int32), "cache": s["cache"]}


def _allowed(mask, v):
    return (torch.bitwise_right_shift(mask[:, :, None], torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(1)[:, :v] != 0


def _plain_edit(s):
    case = s["case"]
    seqs, n, v = case["seqs"], case["rows"], case["vocab"]
    rows, x = seqs * n, s["logits"]
    counts = torch.zeros((rows, v), device="cuda")
    at = torch.arange(case["history"], device="cuda")
    if case["history"]:
        # (the rows of a tree share their sequence's history)
        used = (at < (s["ranges"][:, 1] - s["ranges"][:, 0])[:, None]).to(torch.float32)
        counts.scatter_add_(1, s["recent"].long().repeat_interleave(n, 0), used)
    if n > 1:
        for i in range(seqs):
            mine = slice(i * n, (i + 1) * n)
            counts[mine].scatter_add_(1, s["tokens"][mine].long().expand(n, n), _ancestors(s["parent"][mine]).float())
    hit = counts > 0
    rep, freq, pres = (s[name][:, None] for name in ("repetition", "frequency", "presence"))
    x = torch.where(hit, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * counts
    x = torch.where(hit, x - pres, x)
    if case["biases"]:
        row = torch.arange(rows, device="cuda").repeat_interleave(case["biases"])
        bias = torch.zeros_like(x)
        bias[row, s["bias_id"].long()] = s["bias"]
        x = x + bias
    if case["masks"]:
        ok = _allowed(s["mask"], v)[s["mask_of"].long().clamp(min=0)] | (s["mask_of"] < 0)[:, None]
        x = torch.where(ok, x, -math.inf)
    return {"logits": x}


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


def _own(s):
    fh, ctx = _framework()
    case = s["case"]
    if case["kind"] == "edit":
        if "edit" not in s:
            s["edit"] = fh.LogitsEdit(recent=s["recent"], ranges=s["ranges"], repetition=s["repetition"],
                                      frequency=s["frequency"], presence=s["presence"], parent=s.get("parent"),
                                      tokens=s.get("tokens"), seqs=case["seqs"], bias_off=s.get("bias_off"),
                                      bias_id=s.get("bias_id"), bias=s.get("bias"), mask=s.get("mask"),
                                      mask_of=s.get("mask_of"), masks=case["masks"])
        fh.logits_edit_async(ctx, s["logits"], case["seqs"] * case["rows"], case["vocab"], s["edit"], s["out"])
        return {"logits": s["out"]}
    n_heads, n_kv, hd, rope = MODELS[case["model"]]
    seqs, rows, total = case["seqs"], case["rows"], s["total"]
    if case["kind"] == "accept":
        fh.tree_accept_async(ctx, s["parent"], s["tokens"], s["chosen"], total, s["off"], seqs, rows, s["len"],
                             s["planes"], 2 * case["layers"], n_kv * hd, s["cap"], s["path"], s["count"], s["next"],
                             s["new_len"])
        return {"path": s["path"], "count": s["count"], "next": s["next"], "new_len": s["new_len"], "cache": s["cache"]}
    before = (ctx, s["qkv"], (n_heads + 2 * n_kv) * hd, total, n_heads, n_kv, hd, s["k"], s["v"], seqs, s["cap"],
              s["off"], rows, s["len"], case["len"] + rows)
    turn = (hd if rope else 0, ROPE_BASE, fh.ROPE_NORM if rope == "norm" else fh.ROPE_NEOX, None, 1.0)
    if case["kind"] == "tree":
        fh.gqa_attention_rope_tree_async(*before, s["parent"], None, *turn, s["out"])
    else:
        fh.gqa_attention_rope_prefill_async(*before, None, *turn, s["out"])
    return {"out": s["out"], "k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    return _plain_edit(state) if kind == "edit" else _plain_accept(state) if kind == "accept" else _plain_attention(state)


# ---- from the definitions, in 64 bits ----------------------------------------


def _exact_edit(s):
    case = s["case"]
    n, v = case["rows"], case["vocab"]
    recent, ranges = s["recent"].flatten().tolist(), s["ranges"].tolist()
    tokens = s["tokens"].tolist() if n > 1 else None
    bias = (s["bias_id"].tolist(), s["bias"].double().tolist()) if case["biases"] else None
    out = s["logits"].double()
    for r in range(out.shape[0]):
        seen = {}
        for x in recent[ranges[r][0]:ranges[r][1]]:
            seen[x] = seen.get(x, 0) + 1
        if tokens:
            for t in _path(_parents(n, r // n), r % n):
                x = tokens[r - r % n + t]
                seen[x] = seen.get(x, 0) + 1
        rep, freq, pres = (float(s[name][r]) for name in ("repetition", "frequency", "presence"))
        if seen:
            ids = torch.tensor(list(seen), device="cuda")
            times = torch.tensor(list(seen.values()), device="cuda", dtype=torch.float64)
            x = out[r, ids]
            out[r, ids] = torch.where(x > 0, x / rep, x * rep) - (freq * times + pres)
        if bias:
            mine = slice(r * case["biases"], (r + 1) * case["biases"])
            out[r, torch.tensor(bias[0][mine], device="cuda")] += torch.tensor(bias[1][mine], device="cuda", dtype=torch.float64)
        if r < case["masks"]:
            word = s["mask"][r].cpu().numpy().view("<u4")
            ok = torch.from_numpy((word.repeat(32) >> (torch.arange(word.size * 32).numpy() % 32).astype("u4")) & 1)[:v]
            out[r, ok.cuda() == 0] = -math.inf
    return {"logits": out}


def _exact_accept(s):
    case = s["case"]
    lens, news, _ = _sizes(case)
    cache, first = s["cache"].double(), 0
    for i, (at, n) in enumerate(zip(lens, news)):
        parents, p = _parents(n, i), [0]
        tokens, chosen = (s[name][first:first + n].tolist() for name in ("tokens", "chosen"))
        while True:
            fits = [t for t in range(n) if parents[t] == p[-1] and tokens[t] == chosen[p[-1]]]
            if not fits:
                break
            p.append(fits[0])
        for j, t in enumerate(p):
            cache[:, i, at + j] = s["cache"][:, i, at + t].double()
        first += n
    return {"path": None, "count": None, "next": None, "new_len": None, "cache": cache}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "edit":
        return _exact_edit(s)
    if case["kind"] == "accept":
        return _exact_accept(s)
    n_heads, n_kv, hd, rope = MODELS[case["model"]]
    lens, news, _ = _sizes(case)
    group, first = n_heads // n_kv, 0
    caches = {"k": s["k"].double(), "v": s["v"].double()}
    out = torch.empty((s["total"], n_heads * hd), dtype=torch.float64, device="cuda")
    p = torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd
    freq = torch.tensor(ROPE_BASE, dtype=torch.float64, device="cuda").pow(-p).float()
    for i, (at, new) in enumerate(zip(lens, news)):
        x = s["qkv"][first:first + new].double().view(new, -1, hd)
        if case["kind"] == "tree":
            paths = [_path(_parents(new, i), t) for t in range(new)]
            hidden = torch.ones((new, new), dtype=torch.bool)
            for t, up in enumerate(paths):
                hidden[t, up] = False
            hidden, where = hidden.cuda(), at + torch.tensor([len(up) - 1 for up in paths], device="cuda")
        else:
            hidden = torch.ones((new, new), dtype=torch.bool, device="cuda").triu(1)
            where = at + torch.arange(new, device="cuda")
        if rope:
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (where.float()[:, None] * freq).double())
            y = x[:, :n_heads + n_kv]
            parts = y.chunk(2, dim=-1) if rope == "neox" else (y[..., 0::2], y[..., 1::2])
            z = torch.complex(*(part.contiguous() for part in parts)) * turn[:, None]
            y = torch.cat([z.real, z.imag], -1) if rope == "neox" else torch.view_as_real(z).flatten(-2)
            x = torch.cat([y, x[:, n_heads + n_kv:]], dim=1)
        caches["k"][i, at:at + new] = x[:, n_heads:n_heads + n_kv].flatten(1)
        caches["v"][i, at:at + new] = x[:, n_heads + n_kv:].flatten(1)
        for h in range(n_heads):
            g = slice(h // group * hd, (h // group + 1) * hd)
            z = x[:, h] @ caches["k"][i, :at + new, g].T.contiguous() * hd ** -0.5
            z[:, at:].masked_fill_(hidden, -math.inf)
            out[first:first + new, h * hd:(h + 1) * hd] = torch.softmax(z, dim=1) @ caches["v"][i, :at + new, g]
        first += new
    return {"out": out, "k": caches["k"], "v": caches["v"]}
