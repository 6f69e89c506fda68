"""Inverse frequencies of the rotary embedding and the argument checks of qk_norm_rope (no GPU needed)."""
import ctypes as C
import math

import pytest
import torch

import hils_attention_b200 as hb
from hils_attention_b200 import _lib

BAD_ARG, WORKSPACE = -1, -4


def test_plain_and_linear():
    f, s = hb.rope_frequencies(8, base=10000.0)
    assert s == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    g, s = hb.rope_frequencies(8, base=10000.0, scaling="linear", factor=4.0)
    assert s == 1.0 and torch.allclose(g, f / 4, rtol=1e-14, atol=0)
    assert hb.rope_frequencies(0)[0].numel() == 0


def test_ntk_keeps_the_fastest_and_divides_the_slowest():
    f, g = hb.rope_frequencies(64)[0], hb.rope_frequencies(64, scaling="ntk", factor=8.0)[0]
    assert g[0] == f[0] and math.isclose(float(g[-1]), float(f[-1]) / 8, rel_tol=1e-12)
    assert bool((g <= f).all()) and bool((g[1:] < f[1:]).all())


def test_yarn_keeps_fast_pairs_divides_slow_ones_and_blends_between():
    n, factor = 4096, 16.0
    f, _ = hb.rope_frequencies(128)
    g, s = hb.rope_frequencies(128, scaling="yarn", factor=factor, original_length=n)
    turns = f * n / (2 * math.pi)
    ratio = f / g
    assert math.isclose(s, 0.1 * math.log(factor) + 1.0)
    assert bool((ratio[turns > 40] == 1.0).all()) and torch.allclose(ratio[turns < 0.8], torch.tensor(factor, dtype=torch.float64))
    assert bool((ratio[1:] >= ratio[:-1] - 1e-12).all())
    assert hb.rope_frequencies(128, scaling="yarn", factor=1.0)[1] == 1.0


def test_bad_frequencies_are_refused():
    for kw in (dict(rot=7), dict(rot=-2), dict(rot=8, base=1.0), dict(rot=8, factor=0.5), dict(rot=8, scaling="other"), dict(rot=2, scaling="ntk")):
        with pytest.raises(ValueError):
            hb.rope_frequencies(**kw)


def test_shapes_and_types_are_refused():
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16)
    pos, f, w = torch.arange(5), torch.ones(8, dtype=torch.float64), torch.ones(16)
    ok = dict(q=q, k=k, positions=pos, inv_freq=f, q_weight=w, k_weight=w)
    for change, err in ((dict(q=q[0]), ValueError), (dict(k=k[:1]), ValueError), (dict(k=k[..., :8]), ValueError), (dict(k=k.bfloat16()), TypeError),
                        (dict(positions=pos.float()), TypeError), (dict(positions=pos[:4]), ValueError), (dict(positions=pos.expand(3, 5)), ValueError),
                        (dict(inv_freq=torch.ones(9, dtype=torch.float64)), ValueError), (dict(inv_freq=torch.ones(8, dtype=torch.int64)), ValueError),
                        (dict(inv_freq=f.view(2, 4)), ValueError), (dict(q_weight=w[:8]), ValueError), (dict(q_weight=w.bfloat16()), TypeError)):
        with pytest.raises(err):
            hb.qk_norm_rope(**{**ok, **change})
    with pytest.raises(RuntimeError):
        hb.qk_norm_rope(**ok)                                   # not on a GPU
    with pytest.raises(TypeError):
        hb.qk_norm_rope(**{**ok, "q": q.half(), "k": k.half()})


def _call(bwd=False, *, n=2, D=64, rot=64, heads=(4, 2), dtype=1, wdtype=1, weight=0x1000, dw=0x1000, x=0x1000, B=1, L=3, freq=0x1000, pos=0x1000,
          ws=None, ws_bytes=0):
    lib = _lib.load()
    t = (_lib.RopeTensor * 2)()
    for r, h in zip(t, heads):
        r.x = r.out = r.d_out = x
        r.weight, r.d_weight, r.heads = weight, dw, h
    args = [t, n, C.c_void_p(pos), 0, 0, 1, C.c_void_p(freq), rot, B, L, D, 0, 1.0, 1e-6, dtype, wdtype]
    rc = lib.hils_qk_norm_rope_bwd(*args, ws, ws_bytes, None) if bwd else lib.hils_qk_norm_rope_fwd(*args, None)
    return rc, lib.hils_last_error().decode()


def test_the_c_entry_points_refuse_bad_arguments():
    for kw, word in ((dict(n=0), "one or two"), (dict(n=3), "one or two"), (dict(D=63), "even"), (dict(D=258), "at most 256"), (dict(D=0), "even"),
                     (dict(rot=66), "rotated part"), (dict(rot=3), "rotated part"), (dict(rot=-2), "rotated part"), (dict(heads=(4, -1)), "negative"),
                     (dict(dtype=5), "dtype"), (dict(wdtype=5), "weight dtype"), (dict(x=0), "null"), (dict(freq=0), "null"), (dict(pos=0), "null"),
                     (dict(B=-1), "even and at most")):
        for bwd in (False, True):
            rc, err = _call(bwd, **kw)
            assert rc == BAD_ARG and word in err, (kw, bwd, err)
    assert _call(True, dw=0)[0] == BAD_ARG
    assert _call(True)[0] == WORKSPACE and _call(True, ws=C.c_void_p(0x2000), ws_bytes=64)[0] == WORKSPACE
    need = _lib.load().hils_qk_norm_rope_bwd_workspace_bytes(64)
    assert _call(True, ws=C.c_void_p(0x2004), ws_bytes=need)[0] == WORKSPACE
    assert _lib.load().hils_qk_norm_rope_bwd_workspace_bytes(300) == 0
    assert _call(False, L=0)[0] == 0 and _call(False, heads=(0, 0))[0] == 0


def test_the_packed_tensor_is_the_header_s():
    from hils_attention_b200 import ops
    x = list(range(1, 14))
    assert ops._ROPE_TENSOR.pack(*x) == bytes(_lib.RopeTensor(*x))
