"""Bookkeeping of a step over drafted trees on CPU tensors (the row writes replaced by plain indexing), and the argument
checks of the one-call step (no GPU needed)."""
import ctypes as C
import gc
import weakref

import pytest
import torch

from hils_attention_b200 import _lib, ops
from hils_attention_b200.kv_store import PagedKVStore

BAD_ARG, WORKSPACE = -1, -4


class _Store(PagedKVStore):
    def _copy_pages(self, src, dst):
        self.k_pages[:, list(dst)], self.v_pages[:, list(dst)] = self.k_pages[:, list(src)], self.v_pages[:, list(src)]

    def _commit_drafts(self, path):
        k, v, _ = self._drafts
        for b, nodes in enumerate(path.tolist()):
            for i, x in enumerate(n for n in nodes if n >= 0):
                t = int(self.lens[b]) + i
                pg = int(self.page_table[b, t // 64])
                self.k_pages[:, pg, :, t % 64], self.v_pages[:, pg, :, t % 64] = k[:, b, x], v[:, b, x]


def _store(num_pages=12, max_seqs=3, max_pages=4):
    return _Store(num_pages, max_seqs, max_pages, h_kv=2, head_dim=8, h_q=4, dtype=torch.float32, device="cpu", num_layers=2)


def _fill(st):
    for layer in range(st.num_layers):
        for t in st.draft(layer):
            t.copy_(torch.randn(t.shape))


def test_accepted_nodes_become_tokens():
    st = _store()
    a, b, c = st.allocate(60), st.allocate(0), st.allocate(64)
    st.release(b)
    assert st.begin_tree(7) == 64
    assert [len(st.pages_of(x)) for x in (a, b, c)] == [2, 0, 2]
    _fill(st)
    st.accept_tree([[0, 2, 3, 5], [], [1]])
    assert st.completed() == ([a], [5])                        # a: 60 + 4 tokens; the fourth is node 5
    kc = st.chunk_keys(0, [a])
    assert kc.shape == (1, 64, 2, 8) and torch.equal(kc[0, 60:], st.draft(0)[0][a, [0, 2, 3, 5]])
    st.put_chunk_keys(0, [a], torch.ones(1, 4, 8), torch.ones(1, 4))
    k1, v1, _ = (t.clone() for t in st.draft(1))
    st.end_tree()
    assert (st.length(a), st.length(b), st.length(c)) == (64, 0, 65) and st.lens.tolist() == [64, 0, 65]
    assert bool((st.lmk_k[0, a, 0] == 1).all())
    gk, gv = st.gather(c, 1)
    assert torch.equal(gk[64], k1[c, 1]) and torch.equal(gv[64], v1[c, 1])


def test_reserved_pages_are_used_before_new_ones():
    st = _store()
    a = st.allocate(63)
    st.begin_tree(64)                                          # room for 127 tokens
    assert len(st.pages_of(a)) == 2
    _fill(st)
    st.accept_tree([[4]])
    assert st.completed() == ([a], [4])
    st.end_tree()
    free, pages = st.pool.free, st.pages_of(a)
    st.begin_step()                                            # token 64 goes into the page that is there
    assert st.pool.free == free and st.pages_of(a) == pages and st.length(a) == 64
    st.end_step()
    (b,) = st.fork(a)                                          # a fork shares what is full, not what is reserved
    assert st.pages_of(b)[0] == pages[0] and len(st.pages_of(b)) == 2 and st.pages_of(b)[1] != pages[1]
    st.release(a), st.release(b)
    assert st.pool.free == 11


def test_nothing_accepted_and_a_full_tree():
    st = _store()
    a = st.allocate(64)
    st.begin_tree(64)
    st.accept_tree([[]])
    assert st.completed() == ([], [])
    st.end_tree()
    assert st.length(a) == 64
    st.begin_tree(64)
    _fill(st)
    st.accept_tree([list(range(64))])
    assert st.completed() == ([a], [63])
    st.end_tree()
    assert st.length(a) == 128


def test_order_of_calls_and_bad_paths():
    st = _store(max_pages=2, num_pages=4)
    a = st.allocate(100)
    for bad in (0, 65):
        with pytest.raises(ValueError):
            st.begin_tree(bad)
    with pytest.raises(MemoryError):
        st.begin_tree(29)                                      # 129 tokens, two pages
    with pytest.raises(RuntimeError):
        st.draft(0)
    st.begin_tree(28)
    for call in (lambda: st.begin_tree(1), st.begin_step, st.end_step, st.end_tree, st.completed, lambda: st.fork(a), st.compact, lambda: st.release(a)):
        with pytest.raises(RuntimeError):
            call()
    for paths in ([], [[0], [1]], [[28]], [[-1]], [[1, 1]], [[2, 1]]):
        with pytest.raises(ValueError):
            st.accept_tree(paths)
    st.accept_tree([[0, 27]])
    with pytest.raises(RuntimeError):
        st.accept_tree([[0]])
    st.end_tree()
    assert st.length(a) == 102
    # a path for a row that is no sequence
    b = st.allocate(0)
    c = None
    st2 = _store()
    x, y = st2.allocate(3), st2.allocate(3)
    st2.release(x)
    st2.begin_tree(4)
    with pytest.raises(ValueError):
        st2.accept_tree([[0], [1]])
    st2.accept_tree([[], [1]])


def _call(*, B=2, n=8, h_q=4, h_kv=2, h_lmk=4, D=64, K=4, N=16, W=128, S=64, stride=20, pages=90, max_len=1000, scale=0.125, dtype=_lib.BF16, ptr=0x1000,
          ws=None, ws_bytes=0):
    lib = _lib.load()
    p = C.c_void_p(ptr)
    rc = lib.hils_decode_tree_paged(p, p, p, p, p, p, p, stride, pages, p, max_len, p, p, None, N, p, None, B, n, h_q, h_kv, h_lmk, D, K, S, W, 0, scale,
                                    dtype, ws, ws_bytes, None)
    return rc, lib.hils_last_error().decode()


def test_the_one_call_step_refuses_bad_arguments():
    for kw, word in ((dict(n=65, W=512), "nodes"), (dict(n=-1), "nodes"), (dict(B=-1), "sequences"), (dict(h_q=5, h_lmk=5), "multiple"), (dict(h_lmk=3), "chunk keys"),
                     (dict(S=32), "64 tokens"), (dict(D=96), "head dimension"), (dict(K=33), "topk"), (dict(K=0), "topk"), (dict(h_q=32, h_lmk=32), "8 query heads"),
                     (dict(W=7), "does not hold"), (dict(N=0), "bad size"), (dict(stride=15), "page table"), (dict(N=14), "chunk keys"), (dict(scale=0.0), "sm_scale"),
                     (dict(dtype=9), "dtype"), (dict(ptr=0), "null"), (dict(ptr=0x1008), "aligned"), (dict(max_len=-1), "bad size")):
        rc, err = _call(**kw)
        assert rc == BAD_ARG and word in err, (kw, err)
    need = _lib.load().hils_decode_tree_paged_workspace_bytes(2, 8, 4, 2, 4, 64, 4, 16, 1000, 128, 0, _lib.BF16)
    assert need > 0 and need % 256 == 0
    for ws, size in ((None, 0), (C.c_void_p(0x2000), need - 1), (C.c_void_p(0x2008), need)):
        assert _call(ws=ws, ws_bytes=size)[0] == WORKSPACE
    assert _call(B=0)[0] == 0 and _call(n=0)[0] == 0


def test_shapes_and_types_are_refused():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    ok = dict(q=torch.zeros(2, 3, 4, 64), lmk_q=torch.zeros(2, 3, 4, 64), k_new=torch.zeros(2, 3, 2, 64), v_new=torch.zeros(2, 3, 2, 64),
              k_pages=torch.zeros(5, 2, 64, 64), v_pages=torch.zeros(5, 2, 64, 64), page_table=i32(2, 4), lens=i32(2), max_len=100, parents=i32(2, 3),
              lmk_k=torch.zeros(2, 4, 4, 64), prior_b=None, topk=4)
    for change, err in ((dict(lmk_q=torch.zeros(2, 3, 2, 64)), ValueError), (dict(k_new=torch.zeros(2, 4, 2, 64)), ValueError), (dict(lens=i32(3)), ValueError),
                        (dict(lmk_k=torch.zeros(3, 4, 4, 64)), ValueError), (dict(prior_b=torch.zeros(2, 4, 2)), ValueError), (dict(parents=i32(2, 3).long()), TypeError),
                        (dict(lmk_k=torch.zeros(2, 4, 4, 64).bfloat16()), TypeError), (dict(q=torch.zeros(2, 4, 3, 64).transpose(1, 2)), ValueError)):
        with pytest.raises(err):
            ops.decode_tree_paged(**{**ok, **change})
    with pytest.raises(RuntimeError):
        ops.decode_tree_paged(**ok)                            # not on a GPU


def test_the_drafts_do_not_move_until_a_wider_tree_comes():
    st = _store()
    a, b = st.allocate(3), st.allocate(5)

    def step(n):
        st.begin_tree(n)
        assert all(t.shape[:3] == (2, st.batch, n) and t.is_contiguous() for t in st._drafts)
        at = [t.data_ptr() for t in st._drafts]
        st.accept_tree([[]] * st.batch)
        st.end_tree()
        return at
    first = step(9)
    assert step(4) == first and step(9) == first
    st.release(b)
    assert step(9) == first
    c = st.allocate(1)
    st.fork(a)
    assert c == b and st.batch == 3 and step(9) == first           # all slots
    step(10)
    assert st.lens.tolist() == [3, 1, 3]


def test_sizes_past_32_bits_are_refused():
    """They would reach the library with their upper bits cut off."""
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    ok = dict(q=torch.zeros(2, 3, 4, 64), k_new=torch.zeros(2, 3, 2, 64), v_new=torch.zeros(2, 3, 2, 64), k_pages=torch.zeros(5, 2, 64, 64),
              v_pages=torch.zeros(5, 2, 64, 64), page_table=i32(2, 4), lens=i32(2), max_len=100, parents=i32(2, 3))
    step = dict(ok, lmk_q=ok["q"], lmk_k=torch.zeros(2, 4, 2, 64), prior_b=None, topk=2)
    for change in (dict(window_size=2 ** 32 + 1), dict(max_len=2 ** 32 + 1)):
        with pytest.raises(ValueError, match="max_len"):
            ops.tree_attn_paged(**{**ok, **change})
        with pytest.raises(ValueError, match="max_len"):
            ops.decode_tree_paged(**{**step, **change})
    for topk in (0, -1, 2 ** 32 + 1):
        with pytest.raises(ValueError, match="topk"):
            ops.decode_tree_paged(**{**step, "topk": topk})


def _core_step(monkeypatch, bytes_of):
    """decode_tree_paged of an attention core over a CPU store with the library call replaced: it records the bound and the
    scratch it is given and wants bytes_of(batch, max_len) of scratch.  Returns (step(store, n, max_len=None, core=0), calls)."""
    from hils_attention_b200 import attention
    calls = []

    def library(q, lmk_q, k, v, kp, vp, table, lens, max_len, parents, lmk_k, prior_b, topk, chunk, window, softmax1, workspace=None, return_indices=False):
        need = bytes_of(q.shape[0], max_len)
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(need, dtype=torch.uint8)
        calls.append((max_len, weakref.ref(workspace)))
        return torch.zeros_like(q), workspace
    monkeypatch.setattr(attention.ops, "decode_tree_paged", library)
    cores = [attention.HiLSAttentionCore(attention.HiLSAttentionConfig(4, 2, 2, 64, 128)).eval() for _ in range(2)]
    for i, c in enumerate(cores):
        c.layer_idx = i

    def step(st, n, max_len=None, core=0):
        st.begin_tree(n)
        q, k = torch.zeros(st.batch, n, 4, 8), torch.zeros(st.batch, n, 2, 8)
        try:
            kw = {} if max_len is None else dict(max_len=max_len)
            cores[core].decode_tree_paged(q, k, k, q, st, torch.full((st.batch, n), -1, dtype=torch.int32), **kw)
        finally:
            st.accept_tree([[]] * st.batch)
            st.end_tree()
    return step, calls


def test_a_captured_step_holds_for_all_lengths_a_sequence_may_reach(monkeypatch):
    """The bound is frozen into the graph, the lengths are not."""
    step, calls = _core_step(monkeypatch, lambda b, t: 16)
    st = _store(max_pages=4)
    st.allocate(100)
    step(st, 3)
    assert calls[-1][0] == 100                                 # eager: the present length
    monkeypatch.setattr(_lib, "capturing", lambda device: True, raising=False)
    step(st, 3)
    assert calls[-1][0] == 256
    step(st, 3, max_len=200)                                   # the caller's bound
    assert calls[-1][0] == 200
    monkeypatch.setattr(_lib, "capturing", lambda device: False)
    for bad in (99, 257, -1):
        with pytest.raises(ValueError, match="max_len"):
            step(st, 3, max_len=bad)


def test_what_a_captured_step_writes_to_stays_allocated(monkeypatch):
    """Scratch and drafts of a captured step outlive larger ones: of a longer cache, a larger batch, a wider tree."""
    step, calls = _core_step(monkeypatch, lambda b, t: 64 * b + t)
    st = _store(num_pages=20, max_pages=4)
    st.allocate(10)
    flag = [True]
    monkeypatch.setattr(_lib, "capturing", lambda device: flag[0], raising=False)
    step(st, 3)
    captured, room = calls[-1][1], [weakref.ref(t) for t in st._draft_room]
    st.allocate(70)
    step(st, 3)                                                # a second captured step, of two sequences
    second = calls[-1][1]
    flag[0] = False
    st.allocate(90)
    for n in (3, 8):
        step(st, n)
        step(st, n, max_len=256)
    larger = calls[-1][1]
    gc.collect()
    assert captured() is not None and second() is not None and second() is not captured()
    assert larger() is st.scratch and larger() is not second() and all(r() is not None for r in room)
    # one that no graph writes to goes when a larger one comes
    st2 = _store()
    st2.allocate(5)
    step(st2, 2)
    first = calls[-1][1]
    step(st2, 2, max_len=100)
    gc.collect()
    assert first() is None


def test_the_layers_share_one_scratch_and_stores_do_not(monkeypatch):
    step, calls = _core_step(monkeypatch, lambda b, t: 64)
    a, b = _store(), _store()
    for st in (a, b):
        st.allocate(5)
        for core in (0, 1):
            step(st, 2, core=core)
    got = [r() for _, r in calls]
    assert got[0] is got[1] is a.scratch and got[2] is got[3] is b.scratch and a.scratch is not b.scratch


def test_drafts_of_another_shape_or_type_are_refused(monkeypatch):
    """They would be spread over heads or sequences, or converted, on their way into the pages."""
    from hils_attention_b200 import attention
    monkeypatch.setattr(attention.ops, "decode_tree_paged", lambda q, *a, **kw: (torch.zeros_like(q), torch.zeros(1, dtype=torch.uint8)))
    core = attention.HiLSAttentionCore(attention.HiLSAttentionConfig(4, 2, 2, 64, 128)).eval()
    st = _store()
    st.allocate(5), st.allocate(70)
    st.begin_tree(3)
    for t in st.draft(0):
        t.fill_(7)
    ok = dict(q=torch.zeros(2, 3, 4, 8), k=torch.zeros(2, 3, 2, 8), v=torch.zeros(2, 3, 2, 8), lmk_q=torch.zeros(2, 3, 4, 8))
    parents = torch.full((2, 3), -1, dtype=torch.int32)
    for name in ok:
        x = ok[name]
        for bad in (x[:, :, :1], x[:1], x[:, :1], x[..., :1], x[0], x[:, :2]):
            with pytest.raises(ValueError, match=f": {name} "):
                core.decode_tree_paged(**{**ok, name: bad}, store=st, parents=parents)
        with pytest.raises(TypeError, match=f": {name} "):
            core.decode_tree_paged(**{**ok, name: x.double()}, store=st, parents=parents)
    assert all(bool((t == 7).all()) for t in st.draft(0))      # nothing was written
    core.decode_tree_paged(**ok, store=st, parents=parents)
