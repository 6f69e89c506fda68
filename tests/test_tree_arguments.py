"""Argument checks of the attention over drafted trees that happen before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

import hils_attention_b200 as hb
from hils_attention_b200 import _lib

BAD_ARG, WORKSPACE = -1, -4


def _call(*, B=2, n=8, h_q=4, h_kv=2, D=64, W=128, S=64, stride=40, pages=90, max_len=2000, scale=0.125, dtype=_lib.BF16, ptr=0x1000, ws=None, ws_bytes=0):
    lib = _lib.load()
    p = C.c_void_p(ptr)
    rc = lib.hils_tree_attn_paged(p, p, p, p, p, p, stride, pages, p, max_len, p, p, p, B, n, h_q, h_kv, D, W, S, 1, 1, scale, dtype, ws, ws_bytes, None)
    return rc, lib.hils_last_error().decode()


def test_the_c_entry_point_refuses_bad_arguments():
    for kw, word in ((dict(n=65), "nodes"), (dict(n=-1), "nodes"), (dict(B=-1), "sequences"), (dict(B=70000), "sequences"), (dict(h_q=5), "multiple"),
                     (dict(h_kv=0), "multiple"), (dict(D=96), "head dimension"), (dict(S=32), "64 tokens"), (dict(W=-1), "window"), (dict(dtype=3), "dtype"),
                     (dict(max_len=-1), "length"), (dict(max_len=2 ** 31 - 1), "length"), (dict(scale=0.0), "sm_scale"), (dict(scale=-1.0), "sm_scale"),
                     (dict(scale=float("nan")), "sm_scale"), (dict(scale=float("inf")), "sm_scale"), (dict(stride=0), "bad size"), (dict(pages=0), "bad size"),
                     (dict(max_len=40 * 64 + 1), "page table"), (dict(ptr=0), "null"), (dict(ptr=0x1008), "aligned")):
        rc, err = _call(**kw)
        assert rc == BAD_ARG and word in err, (kw, err)
    need = _lib.load().hils_tree_attn_paged_workspace_bytes(2, 8, 4, 2, 64, 2000, 0, _lib.BF16)     # many tiles, few CTAs: split
    assert need > 0
    for ws, size in ((None, 0), (C.c_void_p(0x2000), need - 1), (C.c_void_p(0x2004), need)):
        rc, err = _call(W=0, ws=ws, ws_bytes=size)
        assert rc == WORKSPACE and str(need) in err
    assert _call(B=0)[0] == 0 and _call(n=0)[0] == 0
    q = _lib.load().hils_tree_attn_paged_workspace_bytes
    assert q(0, 8, 4, 2, 64, 2000, 128, _lib.BF16) == 0 and q(2, 65, 4, 2, 64, 2000, 128, _lib.BF16) == 0
    assert _lib.load().hils_draft_positions(C.c_void_p(0x1000), C.c_void_p(0x1000), C.c_void_p(0x1000), 1, 65, None) == BAD_ARG
    assert _lib.load().hils_draft_positions(None, None, None, 1, 4, None) == BAD_ARG and _lib.load().hils_draft_positions(None, None, None, 0, 4, None) == 0


def test_shapes_and_types_are_refused():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    ok = dict(q=torch.zeros(2, 3, 4, 64), k_new=torch.zeros(2, 3, 2, 64), v_new=torch.zeros(2, 3, 2, 64), k_pages=torch.zeros(5, 2, 64, 64),
              v_pages=torch.zeros(5, 2, 64, 64), page_table=i32(2, 4), lens=i32(2), max_len=100, parents=i32(2, 3))
    for change, err in ((dict(q=ok["q"][0]), ValueError), (dict(k_new=torch.zeros(2, 4, 2, 64)), ValueError), (dict(v_new=torch.zeros(2, 3, 1, 64)), ValueError),
                        (dict(k_pages=torch.zeros(5, 3, 64, 64)), ValueError), (dict(v_pages=torch.zeros(4, 2, 64, 64)), ValueError),
                        (dict(page_table=i32(3, 4)), ValueError), (dict(lens=i32(3)), ValueError), (dict(parents=i32(2, 4)), ValueError),
                        (dict(parents=torch.zeros(2, 3, dtype=torch.int64)), TypeError), (dict(lens=torch.zeros(2)), TypeError),
                        (dict(q=ok["q"].bfloat16()), TypeError), (dict(q=ok["q"].half()), TypeError), (dict(window_size=0), ValueError),
                        (dict(q=torch.zeros(2, 4, 3, 64).transpose(1, 2)), ValueError), (dict(chunk_size=32), ValueError)):
        with pytest.raises(err):
            hb.tree_attn_paged(**{**ok, **change})
    with pytest.raises(RuntimeError):
        hb.tree_attn_paged(**ok)                               # not on a GPU
    for parents, lens in ((i32(2, 3).long(), i32(2)), (i32(2, 3), i32(3)), (i32(3), i32(3)), (i32(2, 3), i32(2).float())):
        with pytest.raises(ValueError):
            hb.draft_positions(parents, lens)
