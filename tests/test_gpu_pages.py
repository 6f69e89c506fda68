"""Page copies, committed drafts, forked and compacted sequences on the GPU.  Data movement: every comparison is bit-exact.
Needs a B200."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def hb():
    import hils_attention_b200 as pkg
    return pkg


def _status():
    from hils_attention_b200 import _lib
    return _lib.query("hils_take_device_status")


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _pools(layers, pages, h, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(layers, pages, h, 64, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    k[0, 1, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0])       # copied like any other bits
    return k, v


@pytest.mark.parametrize("layers,pages,h,D,dtype,n", [
    (1, 3, 1, 64, BF, 1), (2, 9, 2, 64, BF, 4), (1, 40, 3, 128, F32, 17), (3, 16, 5, 8, BF, 7), (1, 1100, 1, 8, BF, 500), (2, 20, 8, 128, BF, 10)])
def test_copy_pages(hb, layers, pages, h, D, dtype, n):
    k, v = _pools(layers, pages, h, D, dtype)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).tolist()
    dst = perm[:n]
    src = [perm[n + i % (pages - n)] for i in range(n)]            # a page may be copied to several others
    wk, wv = k.clone(), v.clone()
    wk[:, dst], wv[:, dst] = wk[:, src], wv[:, src]
    hb.copy_pages(k, v, src, torch.tensor(dst))
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


def test_copy_pages_of_one_layer_and_of_some_layers(hb):
    k, v = _pools(4, 6, 2, 64, BF)
    wk, wv = k.clone(), v.clone()
    wk[2, 5], wv[2, 5] = wk[2, 1], wv[2, 1]
    hb.copy_pages(k[2], v[2], [1], [5])
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))
    wk[::2, 4], wv[::2, 4] = wk[::2, 0], wv[::2, 0]
    hb.copy_pages(k[::2], v[::2], [0], [4])
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))


def test_copy_pages_past_32_bits_of_offset(hb):
    pages, h, D = 33000, 8, 128                                    # 131,072 bytes a page: 4.3 GB
    k = torch.zeros(pages, h, 64, D, dtype=BF, device="cuda")
    k[pages - 2] = 3.0
    k[5] = 7.0
    hb.copy_pages(k, k.clone(), [pages - 2, 5], [1, pages - 1])
    assert bool((k[1] == 3.0).all()) and bool((k[pages - 1] == 7.0).all()) and bool((k[2] == 0).all())


def test_copy_pages_on_another_stream_and_in_a_graph(hb):
    k, v = _pools(2, 8, 2, 64, BF)
    wk = k.clone()
    wk[:, [4, 5]] = wk[:, [1, 1]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        hb.copy_pages(k, v, [1, 1], [4, 5])
    s.synchronize()
    assert torch.equal(_bits(k), _bits(wk))
    src, dst = [1], [6]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hb.copy_pages(k, v, src, dst)
    src[0], dst[0] = 2, 3                                          # a replay copies what was captured
    wk[:, 6] = wk[:, 1]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(_bits(k), _bits(wk))


def _commit_plain(kd, vd, k, v, table, lens, path):
    for b in range(path.shape[0]):
        for i, node in enumerate(path[b].tolist()):
            if node < 0:
                break
            t = int(lens[b]) + i
            pg = int(table[b, t // 64])
            k[:, pg, :, t % 64], v[:, pg, :, t % 64] = kd[:, b, node], vd[:, b, node]


@pytest.mark.parametrize("layers,B,n,m,h,D,dtype", [
    (1, 1, 1, 1, 1, 64, BF), (2, 3, 8, 8, 2, 64, BF), (1, 4, 64, 64, 3, 128, F32), (3, 2, 17, 5, 5, 8, BF), (16, 8, 16, 16, 8, 128, BF)])
def test_commit_drafts(hb, layers, B, n, m, h, D, dtype):
    g = torch.Generator().manual_seed(n + B)
    lens = torch.tensor([(0, 63, 64, 1, 127, 100, 130, 65)[b] for b in range(B)])
    width = 4
    k, v = _pools(layers, B * width + 1, h, D, dtype, seed=n)
    kd, vd = (torch.randn(layers, B, n, h, D, generator=g).to(dtype).cuda() for _ in range(2))
    table = (torch.randperm(B * width, generator=g) + 1).view(B, width)
    path = torch.full((B, m), -1)
    for b in range(B):
        took = [m, 0, (m + 1) // 2, 1][b % 4]
        path[b, :took] = torch.randperm(n, generator=g)[:took].sort().values
    if B > 1 and m > 1:
        path[1, 1] = 0                                             # behind the end of the path: not read as a node
    wk, wv = k.clone(), v.clone()
    _commit_plain(kd, vd, wk, wv, table, lens, path)
    args = [x.to(torch.int32).cuda() for x in (table, lens, path)]
    hb.commit_drafts(kd, vd, k, v, *args)
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))
    hb.commit_drafts(kd[0], vd[0], k[0], v[0], *args)              # one layer, again: the same rows
    assert torch.equal(_bits(k), _bits(wk)) and torch.equal(_bits(v), _bits(wv))
    assert _status() == 0


def test_commit_drafts_skips_what_is_outside_and_reports_it(hb):
    k, v = _pools(1, 4, 2, 64, BF)
    kd = torch.randn(1, 4, 5, 2, 64, device="cuda").to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    wk = k.clone()
    wk[0, 1, :, 10] = kd[0, 0, 2]
    # a path with an id that is no node ends there; the other sequences: none accepted
    hb.commit_drafts(kd, kd, k, v, i32([[1, 2]] * 4), i32([10] * 4), i32([[2, 5, 3], [-1, 0, 0], [-2, 0, 0], [-1, -1, -1]]))
    assert torch.equal(_bits(k), _bits(wk)) and _status() == 8100001
    # pages outside the pool or the table, a negative length
    hb.commit_drafts(kd, kd, k, v, i32([[1, 4], [1, -1], [1, 2], [1, 2]]), i32([64, 64, 128, -5]), i32([[0], [0], [0], [0]]))
    assert torch.equal(_bits(k), _bits(wk)) and _status() == 8100002 and _status() == 0


def test_forked_sequences_decode_like_their_parent_and_grow_apart(hb):
    """Prefill, fork, decode: the parent and a fork that is fed the same tokens give the same outputs; a fork that is fed
    other tokens leaves the parent's as they were; a compaction in between changes nothing."""
    from hils_attention_b200.kv_store import PagedKVStore
    from tests.test_gpu_chain import _core
    from tests.test_gpu_kv_store import K, S, W, _prefill, _sequence
    hq, hk, D, T0, steps = 4, 2, 64, 300, 40
    core = _core(hq, hk, K, S, W).eval()
    seq, other = _sequence(T0 + steps, hq, hk, D, 31, BF), _sequence(T0 + steps, hq, hk, D, 32, BF)

    def run(n_forks, feeds, compact_at=None):
        store = PagedKVStore(64, 4, 16, hk, D, hq, dtype=BF, device="cuda")
        store.pool.shuffle(3)
        dead = store.allocate(200)
        assert _prefill(core, store, seq, T0) == 1
        kids = store.fork(1, n_forks)
        store.release(dead)
        outs = []
        for t in range(T0, T0 + steps):
            if t == compact_at:
                assert store.compact() > 0
            B = store.batch
            rows = [torch.zeros(B, 1, h, D, dtype=BF, device="cuda") for h in (hq, hk, hk, hq)]
            for slot, src in zip([1] + kids, feeds):
                for dst, x in zip(rows, src):
                    dst[slot] = x[0, t:t + 1]
            store.begin_step()
            outs.append(core.decode_paged(*rows, store)[:, 0].clone())
            store.end_step()
        return torch.stack([o[[1] + kids] for o in outs], 1), store, kids

    with torch.no_grad():
        alone, st0, _ = run(0, [seq])
        many, st, kids = run(2, [seq, seq, other], compact_at=T0 + 20)
    assert torch.equal(many[0], alone[0]) and torch.equal(many[1], alone[0])
    assert not torch.equal(many[2], alone[0])
    k0, v0 = st0.gather(1)
    for b in (1, kids[0]):
        k1, v1 = st.gather(b)
        assert torch.equal(k1, k0) and torch.equal(v1, v0)
    assert torch.equal(st.gather(kids[1])[0][:T0], k0[:T0]) and torch.equal(st.gather(kids[1])[0][T0:], other[1][0, T0:])
    assert _status() == 0
