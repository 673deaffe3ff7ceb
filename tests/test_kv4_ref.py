"""The 4-bit cache's test reference against itself and the header, on the CPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import kv4_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("v", [False, True])
def test_every_channel_has_a_place_of_its_own(hd, v):
    place = ref.v_place if v else ref.k_place
    seen = {place(k, c, hd) for k in range(16) for c in range(hd)}
    assert len(seen) == 16 * hd
    assert {o for o, _ in seen} == set(range(16 * hd // 2)) and {s for _, s in seen} == {0, 4}


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("v", [False, True])
def test_pack_and_unpack_agree(hd, v):
    x = np.random.default_rng(hd).standard_normal((13, hd)).astype(np.float32)
    d, q = ref.quantise(x)
    plane, sc = ref.pack(d, q, 16, v)
    got, lev, scale = ref.unpack(plane, sc, hd, range(13), v)
    assert np.array_equal(lev, q) and np.array_equal(scale, d)
    # half a step, or a whole one at +8 steps, which clamps to 7
    step = np.abs(np.repeat(d.astype(np.float64), 32, axis=1))
    assert (np.abs(got - x) <= step * np.where(q == 15, 1.01, 0.5) + 1e-12).all()


def test_levels_of_edge_blocks():
    x = np.zeros((6, 32), np.float32)
    x[1, 3], x[1, 4] = -2.0, 2.0          # the first of two equal magnitudes sets the sign
    x[2, 0], x[2, 1], x[2, 2] = 8.0, 0.5, 1.5  # d = -1: ties go to even
    x[3, 5] = np.float32(1e6)             # beyond f16: the scale saturates
    x[4, 7] = np.inf
    x[5, 9] = np.float32(1e-9)            # a scale that rounds to zero
    d, q = ref.quantise(x)
    assert d[0] == 0 and (q[0] == 8).all()
    assert d[1] == 0.25 and q[1, 3] == 0 and q[1, 4] == 15 and q[1, 0] == 8
    assert d[2] == -1 and q[2, 0] == 0 and q[2, 1] == 8 and q[2, 2] == 6
    assert d[3] == -65504 and q[3, 5] == 0
    assert np.isnan(d[4]) and (q[4] == 8).all()
    assert d[5] == 0 and (q[5] == 8).all()


def test_struct_layouts_match_the_header(tmp_path):
    import ferrum_hip

    src = tmp_path / "layout.c"
    fields = {"fh_kv4_cache": (ferrum_hip.KV4Cache, ["k", "k_d", "v", "v_d", "pos", "weight", "seqs", "n_kv", "head_dim",
                                                     "capacity"]),
              "fh_attn_score": (ferrum_hip.AttnScore, ["softcap", "d_slopes", "d_pos", "d_first", "d_end"])}
    body = "".join(f'printf("%zu\\n", sizeof({t}));' + "".join(f'printf("%zu\\n", offsetof({t}, {n}));' for n in names)
                   for t, (_, names) in fields.items())
    src.write_text('#include <stdio.h>\n#include "ferrum_hip.h"\nint main(void){' + body + "return 0;}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls, names in fields.values():
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, n if hasattr(cls, n) else n[2:]).offset for n in names]
    assert got == want


def test_no_context_is_refused():
    import ferrum_hip

    L, c = ferrum_hip.lib(), ferrum_hip.KV4Cache(1, 1, 64, 8, 16, 16, 16, 16)
    assert L.fh_kv4_append_async(None, c, None, 0, 0, 1, None, 0, None, None, 0, 1.0, 0, None, 1.0, None) == 2
    assert L.fh_kv4_attention_async(None, c, None, 0, 0, 1, None, 0, None, 0, None, None, None) == 2
    assert L.fh_kv4_weigh_async(None, c, None, 0, 0, 1, None, 0, None, 0, None, None) == 2
    assert L.fh_kv4_evict_async(None, c, c, None, 0, 1, 0, None) == 2
    assert L.fh_kv4_read_async(None, c, None, 0, None, None) == 2
