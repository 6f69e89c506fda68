"""Steps over drafted trees through the paged store, as speculative decoding runs them: positions -> norm and rotation ->
tree step -> accepted path into the pages -> pooled keys of completed chunks, with forks, against the same tokens decoded
one by one.  Needs a B200."""
import pytest
import torch

from tests.test_gpu_chain import _core
from tests.util import check

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
S, K, W = 64, 4, 128


def _status():
    from hils_attention_b200 import _lib
    return _lib.query("hils_take_device_status")


class _Model:
    """Raw (not yet normed and rotated) q, k, v, landmark query of a token: a function of the token's id alone."""

    def __init__(self, hq, hk, D, dtype, seed, ids=512):
        g = torch.Generator(device="cuda").manual_seed(seed)
        mk = lambda h: torch.randn(ids, h, D, generator=g, device="cuda").to(dtype)
        self.q, self.k, self.v, self.l = mk(hq), mk(hk), mk(hk), mk(hq)
        self.w = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(3)]
        import hils_attention_b200 as hb
        self.hb = hb
        self.freq, self.scale = hb.rope_frequencies(D, scaling="yarn", factor=4.0, device="cuda")

    def __call__(self, ids, positions):
        """ids, positions (B, L) -> q, k, v, lmk_q as the attention gets them."""
        q, k = self.hb.qk_norm_rope(self.q[ids], self.k[ids], positions, self.freq, self.w[0], self.w[1], attention_scaling=self.scale)
        l, _ = self.hb.qk_norm_rope(self.l[ids], None, positions, self.freq, self.w[2], attention_scaling=self.scale)
        return q, k, self.v[ids], l


def _prefill(core, store, model, ids):
    T = len(ids)
    q, k, v, l = model(torch.tensor([ids], device="cuda"), torch.arange(T, device="cuda"))
    slot = store.allocate(T)
    if T >= S:
        _, aux = core(q, k, v, l, return_aux=True)
        store.write_prefill(slot, 0, k[0], v[0], aux["lmk_k"][0], aux["prior_b"][0])
    else:
        store.write_prefill(slot, 0, k[0], v[0])
    return slot


def _one_by_one(core, store, model, seqs):
    """Decode the tokens seqs[slot] (equal counts) one at a time; outputs and ids (B, steps, ...)."""
    outs, ids = [], []
    for t in range(len(seqs[0])):
        tok = torch.tensor([[s[t]] for s in seqs], device="cuda")
        pos = torch.tensor([[store.length(b)] for b in range(store.batch)], device="cuda")
        store.begin_step()
        o, i = core.decode_paged(*model(tok, pos), store, return_indices=True)
        store.end_step()
        outs.append(o[:, 0].clone())
        ids.append(i[:, 0].clone())
    return torch.stack(outs, 1), torch.stack(ids, 1)


@pytest.mark.parametrize("hq,hk,D,dtype,max_pages,kw", [
    (4, 2, 64, BF, 16, dict()), (4, 4, 128, BF, 512, dict()), (2, 2, 64, F32, 16, dict()), (8, 2, 128, F32, 16, dict()),
    (4, 2, 64, BF, 16, dict(enable_chunk_pooling=True, enable_softmax1=True))])
def test_drafted_steps_match_decoding_one_by_one(hq, hk, D, dtype, max_pages, kw):
    from hils_attention_b200 import ops
    from hils_attention_b200.kv_store import PagedKVStore
    core = _core(hq, hk, K, S, W, **kw).eval()
    model = _Model(hq, hk, D, dtype, 3)
    g = torch.Generator().manual_seed(11)
    h_lmk = hk if kw.get("enable_chunk_pooling") else hq
    prompts = [torch.randint(0, 512, (t,), generator=g).tolist() for t in (600, 290, 50)]
    steps = 90
    future = [torch.randint(0, 512, (steps,), generator=g).tolist() for _ in range(4)]
    future[3][:20] = future[0][:20]                            # the fork of sequence 0 goes its own way after 20 tokens
    new = lambda: PagedKVStore(96, 4, max_pages, hk, D, hq, h_lmk=h_lmk, dtype=dtype, device="cuda")
    with torch.no_grad():
        plain, spec = new(), new()
        spec.pool.shuffle(1)
        for st in (plain, spec):
            for p in prompts:
                _prefill(core, st, model, p)
            assert st.fork(0) == [3]
        want, want_ids = _one_by_one(core, plain, model, future)
        done, rounds, got, got_ids = [0] * 4, 0, [[] for _ in range(4)], [[] for _ in range(4)]
        while min(done) < steps:
            n = [5, 16, 1, 33][rounds % 4]
            rounds += 1
            ids = torch.randint(0, 512, (4, n), generator=g)
            parents = torch.full((4, n), -2, dtype=torch.int32)
            paths = []
            for b in range(4):
                used = n if b != 1 else (n + 1) // 2          # a smaller tree in one row
                for j in range(used):
                    parents[b, j] = int(torch.randint(-1, j, (1,), generator=g)) if j else -1
                # the true continuation along one random root-to-node line
                line, j = [], int(torch.randint(0, used, (1,), generator=g))
                while j >= 0:
                    line.append(j)
                    j = int(parents[b, j])
                line = line[::-1][:steps - done[b]]
                for d, j in enumerate(line):
                    ids[b, j] = future[b][done[b] + d]
                paths.append(line if rounds % 5 else [])       # now and then nothing is accepted
            spec.begin_tree(n)
            dev = parents.cuda()
            pos = ops.draft_positions(dev, spec.lens[:4])
            o, idx = core.decode_tree_paged(*model(ids.cuda(), pos), spec, dev, return_indices=True)
            assert not bool(o[(dev < -1)].any())               # absent nodes
            spec.accept_tree(paths)
            core.pool_accepted(spec)
            spec.end_tree()
            for b, line in enumerate(paths):
                got[b] += [o[b, j].clone() for j in line]
                got_ids[b] += [idx[b, j].clone() for j in line]
                done[b] += len(line)
        assert plain.lens.tolist() == spec.lens.tolist()
        for b in range(4):
            same = (torch.stack(got_ids[b]) == want_ids[b]).all(-1)                  # (steps, hk)
            assert same.float().mean().item() >= 0.97, f"slot {b}"
            rows = same.repeat_interleave(hq // hk, dim=1)
            check(torch.stack(got[b])[rows], want[b][rows], dtype, f"drafted steps, slot {b}")
            for x, y in zip(spec.gather(b), plain.gather(b)):
                assert torch.equal(x, y)
            c = plain.length(b) // S
            assert torch.equal(spec.lmk_k[0, b, :c], plain.lmk_k[0, b, :c]) and torch.equal(spec.prior_b[0, b, :c], plain.prior_b[0, b, :c])
    assert _status() == 0


def test_nan_drafts_of_rejected_branches_leave_no_trace():
    """A branch of NaN: the other branches' outputs are bit for bit what they are without it, and nothing of it is committed."""
    from hils_attention_b200.kv_store import PagedKVStore
    hq, hk, D = 4, 2, 64
    core, model = _core(hq, hk, K, S, W).eval(), _Model(hq, hk, D, BF, 5)
    parents = torch.tensor([[-1, 0, 0, 1, 2]], dtype=torch.int32, device="cuda")
    outs = []
    with torch.no_grad():
        for spoil in (False, True):
            store = PagedKVStore(32, 1, 16, hk, D, hq, dtype=BF, device="cuda")
            _prefill(core, store, model, list(range(310)))
            store.begin_tree(5)
            x = [t.clone() for t in model(torch.tensor([[1, 2, 3, 4, 5]], device="cuda"), torch.tensor([[310, 311, 311, 312, 312]], device="cuda"))]
            if spoil:
                for t in x:
                    t[:, [2, 4]] = float("nan")
            o = core.decode_tree_paged(*x, store, parents)
            store.accept_tree([[0, 1, 3]])
            core.pool_accepted(store)
            store.end_tree()
            outs.append((o[:, [0, 1, 3]].clone(), *store.gather(0)))
            if spoil:
                assert bool(torch.isnan(o[:, [2, 4]]).all())
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and store.length(0) == 313


def test_a_captured_tree_step_follows_its_inputs():
    from hils_attention_b200 import ops
    hq, hk, D, n, N = 4, 2, 64, 6, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    q, l, k, v, kp, vp = mk(2, n, hq, D), mk(2, n, hq, D), mk(2, n, hk, D), mk(2, n, hk, D), mk(40, hk, 64, D), mk(40, hk, 64, D)
    table = torch.randperm(40)[:32].view(2, 16).to(torch.int32).cuda()
    lens, lmk, pb = torch.tensor([700, 300], dtype=torch.int32, device="cuda"), mk(2, N, hq, D), torch.randn(2, N, hq, generator=g, device="cuda")
    parents = torch.tensor([[-1, 0, 1, 1, 2, -1], [-1, -1, 0, -2, -2, -2]], dtype=torch.int32, device="cuda")
    call = lambda ws=None: ops.decode_tree_paged(q, l, k, v, kp, vp, table, lens, 900, parents, lmk, pb, K, 64, W, workspace=ws)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = call()
    lens.copy_(torch.tensor([301, 890], dtype=torch.int32))
    parents[1, 3] = 2
    q.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, call()[0]) and _status() == 0


@pytest.mark.parametrize("hq,hk,D,h_lmk", [(8, 2, 128, 8), (8, 2, 64, 2), (16, 2, 128, 2)])
def test_grouped_heads_over_more_than_one_range_of_chunks(hq, hk, D, h_lmk):
    """bf16 with room for thousands of chunks streams the chunk keys in ranges of 1024.  A tree of first nodes only: every node
    against the single-token step with its query, key and value."""
    from hils_attention_b200 import ops
    n, N, K8 = 5, 2304, 8
    lengths = [131072 + 70, 65536 + 640, 40000, 300]
    B, width = len(lengths), N
    g = torch.Generator(device="cuda").manual_seed(D + h_lmk)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    pages = sum(t // 64 + 1 for t in lengths) + 1
    order = torch.randperm(pages - 1, generator=torch.Generator().manual_seed(1)).to(torch.int32) + 1
    table, at = torch.zeros(B, width, dtype=torch.int32), 0
    for b, t in enumerate(lengths):
        table[b, :t // 64 + 1] = order[at:at + t // 64 + 1]
        at += t // 64 + 1
    table, lens = table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kp, vp, lmk = mk(pages, hk, 64, D), mk(pages, hk, 64, D), mk(B, N, h_lmk, D)
    pb = torch.randn(B, N, hq, generator=g, device="cuda")
    q, l, k, v = mk(B, n, hq, D), mk(B, n, hq, D), mk(B, n, hk, D), mk(B, n, hk, D)
    parents = torch.full((B, n), -1, dtype=torch.int32, device="cuda")
    o, idx, _ = ops.decode_tree_paged(q, l, k, v, kp, vp, table, lens, max(lengths), parents, lmk, pb, K8, 64, W, return_indices=True)
    far = 0
    for j in range(n):
        want, ids, _ = ops.decode_step_paged(*(x[:, j].contiguous() for x in (q, l, k, v)), kp, vp, table, lens, max(lengths), lmk, pb, K8, 64, W,
                                             return_indices=True)
        far += int((ids[0] >= 1024).sum())
        same = (idx[:, j] == ids).all(-1)                       # the window's log-sum-exp decides none of the ids
        assert bool(same.all()), f"node {j}: {int((~same).sum())} rows selected otherwise"
        check(o[:, j], want, BF, f"node {j}")
    assert far > 0 and _status() == 0


def _random_sequence(store, T, g):
    slot = store.allocate(T)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    store.write_prefill(slot, 0, mk(T, store.h_kv, store.D), mk(T, store.h_kv, store.D), mk(T // S, store.h_lmk, store.D),
                        torch.randn(T // S, store.h_q, generator=g, device="cuda"))
    return slot


def test_a_captured_step_replays_at_lengths_its_capture_did_not_have():
    """Captured while nothing is selectable, replayed past the window and past 1024 selectable chunks (bf16 with room for 512
    chunks or more streams the chunk keys first), with a second batch size captured and longer eager steps in between."""
    from hils_attention_b200.kv_store import PagedKVStore
    hq, hk, D, n = 8, 2, 64, 6
    core = _core(hq, hk, K, S, W).eval()
    store = PagedKVStore(2400, 2, 1152, hk, D, hq, dtype=BF, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    x = [mk(2, n, hq, D), mk(2, n, hk, D), mk(2, n, hk, D), mk(2, n, hq, D)]
    parents = torch.tensor([[-1, 0, 1, 1, 2, -1], [-1, -1, 0, -2, -2, -2]], dtype=torch.int32, device="cuda")

    def call(B, **kw):
        return core.decode_tree_paged(*(t[:B] for t in x), store, parents[:B], return_indices=True, **kw)

    def in_step(f):
        store.begin_tree(n)
        try:
            return f()
        finally:
            store.accept_tree([[]] * store.batch)
            store.end_tree()

    def capture(B):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(B)
        return graph, out
    with torch.no_grad():
        _random_sequence(store, 100, g)
        in_step(lambda: call(1))
        one = in_step(lambda: capture(1))
        _random_sequence(store, 70, g)
        two = in_step(lambda: capture(2))
        store.release(1)
        for T in (110, 150, 700, 9000, 70000):
            store.release(0)
            assert _random_sequence(store, T, g) == 0
            for B, (graph, out) in ((1, one), (2, two)):
                if B == 2:
                    _random_sequence(store, T // 2, g)
                x[0].neg_()

                def compare():
                    want = [t.clone() for t in call(B, max_len=store.max_pages * S)]
                    plain = [t.clone() for t in call(B)]                    # the present lengths: the same selection
                    for t in out:
                        t.zero_()
                    graph.replay()
                    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), f"{T} tokens, batch {B}"
                    assert torch.equal(plain[1], want[1])
                    return want
                o, idx = in_step(compare)
                if T >= 70000:
                    assert int(idx.max()) >= 1024
            store.release(1)
    assert _status() == 0


def test_a_length_past_the_bound_is_reported_and_selects_from_written_scores_only():
    """What a graph does whose sequence has outgrown the bound of its capture: the scores behind the bound are not computed."""
    from hils_attention_b200 import ops
    hq, hk, D, n, N, T, bound = 4, 2, 64, 3, 1200, 70000, 1000
    g = torch.Generator(device="cuda").manual_seed(6)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    kp, vp, lmk = mk(1100, hk, 64, D), mk(1100, hk, 64, D), mk(1, N, hq, D)
    table = torch.zeros(1, N, dtype=torch.int32, device="cuda")
    table[0, :1099] = torch.arange(1, 1100, dtype=torch.int32)
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    q, l, k, v = mk(1, n, hq, D), mk(1, n, hq, D), mk(1, n, hk, D), mk(1, n, hk, D)
    parents = torch.tensor([[-1, 0, 1]], dtype=torch.int32, device="cuda")
    call = lambda max_len, ws=None: ops.decode_tree_paged(q, l, k, v, kp, vp, table, lens, max_len, parents, lmk, None, K, 64, W, workspace=ws, return_indices=True)
    full, ids, ws = call(T)
    assert int(ids.max()) > bound // 64 and _status() == 0
    for fill in (0x50, 0xd0, 0xff):                            # large scores, small ones, NaN
        ws.fill_(fill)
        o, ids, again = call(bound, ws)
        assert again is ws and _status() == 8200003
        assert int(ids.min()) >= 0 and int(ids.max()) < (bound + n - 1 - W + 1) // 64
        assert bool(torch.isfinite(o).all())
    for fill in (0x50, 0xff):                                  # the single-token step reads the same scores
        one = torch.full((ws.numel(),), fill, dtype=torch.uint8, device="cuda")
        _, ids, again = ops.decode_step_paged(q[:, 0].contiguous(), l[:, 0].contiguous(), k[:, 0].contiguous(), v[:, 0].contiguous(), kp, vp, table, lens, bound,
                                              lmk, None, K, 64, W, workspace=one, return_indices=True)
        assert again is one and int(ids.min()) >= 0 and int(ids.max()) < (bound - W + 1) // 64
    o, ids, _ = call(T, ws)
    assert torch.equal(o, full) and _status() == 0


def test_a_store_stays_on_its_device():
    """A store made on "cuda" is on the device that was current then, and so is all it makes later."""
    from hils_attention_b200.kv_store import PagedKVStore
    store = PagedKVStore(8, 2, 4, 2, 64, 4, device="cuda")
    assert store.device == store.k_pages.device and store.device.index is not None
    store.allocate(10)
    store.begin_tree(3)
    assert all(t.device == store.device for t in store.draft(0))
    store.accept_tree([[0]])
    store.end_tree()
    assert store.lens.tolist() == [11, 0]
