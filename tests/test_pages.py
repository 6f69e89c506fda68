"""Forking, compacting and freeing pages of the paged store: bookkeeping on CPU tensors, with the page copy itself replaced
by an index assignment, and the argument checks that happen before anything is launched."""
import ctypes as C

import pytest
import torch

from hils_attention_b200 import _lib, ops
from hils_attention_b200.kv_store import PagedKVStore, PagePool

BAD_ARG = -1


class _Store(PagedKVStore):
    def _copy_pages(self, src, dst):
        self.k_pages[:, list(dst)] = self.k_pages[:, list(src)]
        self.v_pages[:, list(dst)] = self.v_pages[:, list(src)]


def _store(num_pages=24, max_seqs=5, max_pages=6, layers=2):
    return _Store(num_pages, max_seqs, max_pages, h_kv=2, head_dim=8, h_q=4, dtype=torch.float32, device="cpu", num_layers=layers)


def _fill(st, T, seed):
    g = torch.Generator().manual_seed(seed)
    slot = st.allocate(T)
    n = T // 64
    kv = []
    for layer in range(st.num_layers):
        k, v = torch.randn(T, 2, 8, generator=g), torch.randn(T, 2, 8, generator=g)
        lk, pb = torch.randn(n, 4, 8, generator=g), torch.randn(n, 4, generator=g)
        st.write_prefill(slot, layer, k, v, lk if n else None, pb if n else None)
        kv.append((k, v, lk, pb))
    return slot, kv


def _holds(st, slot, kv):
    for layer, (k, v, lk, pb) in enumerate(kv):
        gk, gv = st.gather(slot, layer)
        n = lk.shape[0]
        if not (torch.equal(gk, k) and torch.equal(gv, v) and torch.equal(st.lmk_k[layer, slot, :n], lk)
                and torch.equal(st.prior_b[layer, slot, :n], pb)):
            return False
    return True


@pytest.mark.parametrize("T", [0, 1, 63, 64, 65, 130, 192])
def test_fork_shares_full_pages_and_copies_the_last_one(T):
    st = _store()
    a, kv = _fill(st, T, T)
    free = st.pool.free
    kids = st.fork(a, 3)
    assert kids == [1, 2, 3] and st.batch == 4
    assert st.pool.free == free - (3 if T % 64 else 0)
    for b in kids:
        assert st.length(b) == T and _holds(st, b, kv)
        assert st.pages_of(b)[:T // 64] == st.pages_of(a)[:T // 64]
        assert st.page_table[b, :len(st.pages_of(b))].tolist() == st.pages_of(b)
    tails = [st.pages_of(b)[T // 64] for b in [a] + kids if T % 64]
    assert len(set(tails)) == len(tails)
    # the parent goes, the children stay
    st.release(a)
    assert all(_holds(st, b, kv) for b in kids)
    for b in kids:
        st.release(b)
    assert st.pool.free == 23 and st.batch == 0


def test_forked_sequences_grow_apart():
    st = _store()
    a, _ = _fill(st, 127, 1)
    (b,) = st.fork(a)
    for _ in range(3):                          # both fill their last page and take one of their own
        st.begin_step()
        st.end_step()
    assert st.pages_of(a)[0] == st.pages_of(b)[0] and not set(st.pages_of(a)[1:]) & set(st.pages_of(b)[1:])
    assert st.length(a) == st.length(b) == 130


def test_fork_that_does_not_fit_changes_nothing():
    st = _store(num_pages=5, max_seqs=3)
    a, kv = _fill(st, 130, 2)                   # three of four pages
    with pytest.raises(MemoryError):
        st.fork(a, 2)                           # two tails, one page left
    with pytest.raises(MemoryError):
        st.fork(a, 3)                           # no third slot
    assert st.batch == 1 and st.pool.free == 1 and _holds(st, a, kv)
    with pytest.raises(ValueError):
        st.fork(1)
    with pytest.raises(ValueError):
        st.fork(a, -1)
    assert st.fork(a, 0) == []
    st.begin_step()
    with pytest.raises(RuntimeError):
        st.fork(a)
    with pytest.raises(RuntimeError):
        st.compact()
    st.end_step()


def test_a_prefill_into_shared_pages_is_refused():
    st = _store()
    a, kv = _fill(st, 64, 3)
    (b,) = st.fork(a)
    with pytest.raises(RuntimeError):
        st.write_prefill(b, 0, torch.zeros(64, 2, 8), torch.zeros(64, 2, 8))
    assert _holds(st, a, kv)


def test_compact_moves_the_pages_in_use_to_the_front():
    st = _store(num_pages=40, max_seqs=6)
    st.pool.shuffle(5)
    seqs = dict(_fill(st, T, 10 + T) for T in (130, 64, 300, 5))
    kid = st.fork(2)[0]
    seqs[kid] = seqs[2]
    st.release(1)
    del seqs[1]
    used = 39 - st.pool.free
    moved = st.compact()
    assert moved > 0 and st.compact() == 0
    pages = sorted({p for b in seqs for p in st.pages_of(b)})
    assert pages == list(range(1, used + 1)) and st.pool.free == 39 - used
    for b, kv in seqs.items():
        assert _holds(st, b, kv) and st.page_table[b, :len(st.pages_of(b))].tolist() == st.pages_of(b)
    for b in list(seqs):
        st.release(b)
    assert st.pool.free == 39 and sorted(st.pool.take(39)) == list(range(1, 40))


def test_pool_counts_the_holders_of_a_page():
    pool = PagePool(4)
    a, b = pool.take(2)
    pool.share([a])
    assert pool.shared(a) and not pool.shared(b)
    pool.give([a])
    assert pool.free == 1 and not pool.shared(a)
    pool.give([a, b])
    assert pool.free == 3
    with pytest.raises(ValueError):
        pool.give([a])
    with pytest.raises(ValueError):
        pool.share([a])
    with pytest.raises(ValueError):
        pool.share([0])


# ---- argument checks -------------------------------------------------------------------------------------------------
def _copy(src, dst, *, layers=1, pages=8, layer_bytes=8 * 1024, page_bytes=1024, ptr=0x1000, n=None):
    lib = _lib.load()
    s, d = (C.c_int32 * max(1, len(src)))(*src), (C.c_int32 * max(1, len(dst)))(*dst)
    rc = lib.hils_copy_pages(C.c_void_p(ptr), C.c_void_p(ptr), s, d, len(src) if n is None else n, layers, pages, layer_bytes, page_bytes, None)
    return rc, lib.hils_last_error().decode()


@pytest.mark.parametrize("src,dst,word", [
    ([8], [1], "outside"), ([-1], [1], "outside"), ([1], [8], "outside"), ([1], [-1], "outside"), ([2 ** 31 - 1], [1], "outside"),
    ([1, 2], [3, 3], "written twice"), ([1, 3], [3, 4], "read and written"), ([1], [1], "read and written"),
    ([1, 2], [2, 1], "read and written")])
def test_copy_pages_refuses_bad_pairs(src, dst, word):
    rc, err = _copy(src, dst)
    assert rc == BAD_ARG and word in err


def test_copy_pages_refuses_bad_sizes():
    for kw, word in ((dict(page_bytes=1000), "multiple of 16"), (dict(page_bytes=0), "multiple of 16"), (dict(layers=2, layer_bytes=4096), "do not hold"),
                     (dict(pages=0), "no pages"), (dict(ptr=0), "null"), (dict(ptr=0x1008), "aligned"), (dict(n=-1), "negative"),
                     (dict(layers=40000), "layers")):
        rc, err = _copy([1], [2], **kw)
        assert rc == BAD_ARG and word in err, kw
    assert _copy([], [])[0] == 0 and _copy([1], [2], layers=0)[0] == 0


def test_copy_pages_takes_its_ids_from_the_host():
    k = torch.zeros(2, 8, 2, 64, 8)
    for src, dst, err in (([1, 2], [3], ValueError), (torch.tensor([1.0]), [2], TypeError), (torch.tensor([2 ** 32 + 1]), [2], ValueError),
                          (torch.tensor([[1]]), [2], ValueError)):
        with pytest.raises(err):
            ops.copy_pages(k, k, src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages(k, k[:1], [1], [2])
    with pytest.raises(ValueError):
        ops.copy_pages(k[0, 0], k[0, 0], [1], [2])
    with pytest.raises(ValueError):
        ops.copy_pages(k.transpose(2, 3), k.transpose(2, 3), [1], [2])
    with pytest.raises(RuntimeError):
        ops.copy_pages(k, k, [1], [2])          # not on a GPU
    ops.copy_pages(k, k, [], [])


def _commit(*, layers=1, B=2, n=4, m=4, h_kv=2, D=64, stride=3, pages=8, layer_bytes=8 * 64 * 2 * 64 * 2, dtype=_lib.BF16, ptr=0x1000):
    p = C.c_void_p(ptr)
    lib = _lib.load()
    rc = lib.hils_commit_drafts(p, p, p, p, p, stride, pages, p, p, layers, B, n, m, h_kv, D, layer_bytes, dtype, None)
    return rc, lib.hils_last_error().decode()


def test_commit_drafts_refuses_bad_sizes():
    for kw, word in ((dict(m=5), "path of 5"), (dict(D=4), "multiple of 16"), (dict(h_kv=0), "non-positive"), (dict(pages=0), "non-positive"),
                     (dict(stride=0), "non-positive"), (dict(layers=2, layer_bytes=64), "do not hold"), (dict(dtype=7), "dtype"),
                     (dict(ptr=0), "null"), (dict(ptr=0x1004), "aligned"), (dict(B=-1), "path"), (dict(layers=70000), "too many")):
        rc, err = _commit(**kw)
        assert rc == BAD_ARG and word in err, (kw, err)
    assert _commit(B=0)[0] == 0 and _commit(m=0)[0] == 0 and _commit(layers=0)[0] == 0


def test_commit_drafts_checks_shapes_and_types():
    kd, kp = torch.zeros(2, 3, 4, 2, 8), torch.zeros(2, 8, 2, 64, 8)
    tab, lens, path = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32)
    ok = dict(k_draft=kd, v_draft=kd, k_pages=kp, v_pages=kp, page_table=tab, lens=lens, path=path)
    for change, err in ((dict(k_draft=kd[0]), ValueError), (dict(k_draft=kd[:1], v_draft=kd[:1]), ValueError), (dict(v_draft=kd.bfloat16()), TypeError),
                        (dict(path=path.long()), TypeError), (dict(path=torch.zeros(3, 5, dtype=torch.int32)), ValueError),
                        (dict(lens=lens[:2]), ValueError), (dict(path=path[:, ::2]), ValueError), (dict(page_table=tab[:2]), ValueError),
                        (dict(k_draft=kd.transpose(1, 2), v_draft=kd.transpose(1, 2)), ValueError)):
        with pytest.raises(err):
            ops.commit_drafts(**{**ok, **change})
    with pytest.raises(RuntimeError):
        ops.commit_drafts(**ok)                 # not on a GPU


def test_copy_pages_does_not_round_or_cut_page_ids():
    k = torch.zeros(2, 8, 2, 64, 8)
    for src, err in (([1.7], TypeError), ([1, 2.5], TypeError), ([2 ** 32 + 1], ValueError), ([-2 ** 31 - 1], ValueError), ([2 ** 70], ValueError), ([[1]], TypeError)):
        with pytest.raises(err):
            ops.copy_pages(k, k, src, [2] * len(src))
        with pytest.raises(err):
            ops.copy_pages(k, k, [2] * len(src), src)
    for none in ([], (), range(0), torch.empty(0, dtype=torch.int64)):
        ops.copy_pages(k, k, none, [])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.copy_pages(k, k, range(1, 3), (3, 4))


def test_strides_of_dimensions_of_one_do_not_matter():
    """One head, one page, one layer: a view that is contiguous with other strides there is a pool like any other."""
    head = torch.zeros(3, 64, 1, 8).transpose(1, 2)                            # (3, 1, 64, 8)
    page = torch.zeros(2, 1, 2, 64, 8).as_strided((2, 1, 2, 64, 8), (1024, 7, 512, 8, 1))
    layer = torch.zeros(1, 3, 2, 64, 8).as_strided((1, 3, 2, 64, 8), (5, 1024, 512, 8, 1))
    for k in (head, page, layer):
        assert k.is_contiguous()
        v = torch.zeros(k.shape)
        if k.shape[-4] > 1:
            for pools in ((k, v), (v, k)):
                with pytest.raises(RuntimeError, match="CUDA"):                # past the checks
                    ops.copy_pages(*pools, [1], [2])
        assert ops._pool_layers(k, v, "pools") == ops._pool_layers(v, k, "pools") == ops._pool_layers(v, v, "pools")
    some = torch.zeros(4, 3, 2, 64, 8)[::2]
    assert ops._pool_layers(some, some, "pools") == (2, 3, 2 * 3 * 1024 * 4)
    for k, v in ((some, torch.zeros(2, 3, 2, 64, 8)), (torch.zeros(2, 3, 64, 2, 8).transpose(2, 3),) * 2, (torch.zeros(3, 64, 2, 8).transpose(1, 2),) * 2):
        with pytest.raises(ValueError):
            ops.copy_pages(k, v, [1], [2])
