"""Attention of drafted trees over the paged store against the definition in 64 bits.  Needs a B200.

Tolerances.  A score is a sum of D products in fp32, off by at most d = scale * (D + 8) * 2^-24 * max_j sum_i |q_i k_ji| (plus a
relative 2^-22 for the exponential's argument); a weight is then off by a relative 2 d, an output by 4 d max|v|, and lse by d plus
its own rounding.  In bf16 the weights are rounded to half a step, 2^-8 relative, before they meet the values: 2^-8 sum_j p_j |v_j|
more (the row sum is not rounded), and the output is rounded once more, 2^-8 |o|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def hb():
    import hils_attention_b200 as pkg
    return pkg


def _status():
    from hils_attention_b200 import _lib
    return _lib.query("hils_take_device_status")


def _lines(parents):
    """Node by node the list of itself and its ancestors from the root on; [] for an absent node."""
    out = []
    for j, p in enumerate(parents):
        if p == -1:
            out.append([j])
        elif 0 <= p < j and out[p]:
            out.append(out[p] + [j])
        else:
            out.append([])
    return out


def _reference(q, k, v, kp, vp, table, lens, parents, W, mask_lmk, expand, scale):
    """(o, lse, sum p|v|, d, max|v| seen) in 64 bits on the CPU, row by row from the definition."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    B, n, hq, D = q.shape
    G = hq // k.shape[2]
    o, pv = torch.zeros(B, n, hq, D, dtype=torch.float64), torch.zeros(B, n, hq, D, dtype=torch.float64)
    lse = torch.full((B, n, hq), -INF, dtype=torch.float64)
    d, top = torch.zeros(B, n, hq, dtype=torch.float64), torch.zeros(B, n, hq, dtype=torch.float64)
    for b in range(B):
        T = int(lens[b])
        ids = table[b, :(T + 63) // 64].long().to(kp.device)
        ck, cv = (x[ids].transpose(1, 2).reshape(-1, k.shape[2], D)[:T].double().cpu() for x in (kp, vp))
        lines = _lines(parents[b].tolist())
        at = [T + len(line) - 1 for line in lines]
        for j, line in enumerate(lines):
            if not line:
                continue
            lo = -INF if W is None else at[j] - W + 1
            if W is not None and expand:
                lo = lo // 64 * 64
            old = [s for s in range(T) if s >= lo and not (mask_lmk and s % 64 == 63)]
            new = [i for i in line if at[i] >= lo and not (mask_lmk and at[i] % 64 == 63)]
            if not old and not new:
                continue
            keys, vals = torch.cat((ck[old], k[b, new])), torch.cat((cv[old], v[b, new]))        # (m, h_kv, D)
            for h in range(hq):
                kk, vv = keys[:, h // G], vals[:, h // G]
                s = kk @ q[b, j, h] * scale
                lse[b, j, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                o[b, j, h], pv[b, j, h] = p @ vv, p @ vv.abs()
                d[b, j, h] = scale * (D + 8) * 2.0 ** -24 * float((kk.abs() @ q[b, j, h].abs()).max()) + 2.0 ** -22 * float(s.abs().max())
                top[b, j, h] = float(vv.abs().max())
    return o, lse, pv, d, top


def _near(got, ref, dtype, what=""):
    (o, lse), (ro, rl, pv, d, top) = got, ref
    tol = 4 * d[..., None] * top[..., None] + (2.0 ** -8 * (pv + ro.abs()) if dtype == BF else 2.0 ** -23 * (pv + ro.abs()))
    eo, el = (o.double().cpu() - ro).abs(), lse.double().cpu()
    assert o.dtype == dtype and lse.dtype == F32
    assert torch.equal(torch.isneginf(el), torch.isneginf(rl)), f"{what}: rows that see nothing differ"
    assert bool((eo <= tol).all()), f"{what}: o off by {float((eo - tol).max()):.3e} over the bound, worst {float(eo.max()):.3e}"
    fin = ~torch.isneginf(rl)
    le = (el - rl).abs()[fin]
    assert bool((le <= d[fin] + 1e-6 * (1 + rl[fin].abs())).all()), f"{what}: lse off by {float(le.max()):.3e}"


def _tree(kind, n, g):
    if kind == "chain":
        return [j - 1 for j in range(n)]
    if kind == "star":
        return [-1] * n
    if kind == "binary":
        return [(j - 1) // 2 for j in range(n)]
    if kind == "random":
        return [int(torch.randint(-1, j, (1,), generator=g)) if j else -1 for j in range(n)]
    if kind == "short":                                       # a shorter tree in a batch
        m = max(1, n // 2)
        return [max(j - 2, -1) for j in range(m)] + [-2] * (n - m)
    if kind == "broken":                                      # parents that are no earlier node, and what hangs from them
        p = [j - 1 for j in range(n)]
        for j, x in ((1, 1), (4, 9), (6, -3), (8, 2 ** 30), (11, -2 ** 31)):
            if j < n:
                p[j] = x
        return p
    if kind == "none":
        return [-2] * n
    raise KeyError(kind)


def _problem(B, n, hq, hk, D, dtype, lens, kinds, seed=0, spare=3, stride=None):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gd, device="cuda").to(dtype)
    need = [(t + 63) // 64 for t in lens]
    width = stride or max(max(need), 1) + 1
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((B, width), -7, dtype=torch.int32)     # entries past a sequence's last chunk are not read
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]].to(torch.int32)
        at += need[b]
    parents = torch.tensor([_tree(kinds[b % len(kinds)], n, g) for b in range(B)], dtype=torch.int32)
    kp, vp = mk(pages, hk, 64, D), mk(pages, hk, 64, D)
    # what lies behind a sequence's last token and in the pages of nobody may be anything
    for x in order[at:].tolist():
        kp[x], vp[x] = NAN, INF
    for b in range(B):
        if lens[b] % 64:
            kp[int(table[b, need[b] - 1]), :, lens[b] % 64:], vp[int(table[b, need[b] - 1]), :, lens[b] % 64:] = INF, NAN
    return dict(q=mk(B, n, hq, D), k=mk(B, n, hk, D), v=mk(B, n, hk, D), kp=kp, vp=vp, table=table, lens=torch.tensor(lens, dtype=torch.int32),
                parents=parents)


def _call(hb, p, W=None, max_len=None, workspace=None, **kw):
    return hb.tree_attn_paged(p["q"], p["k"], p["v"], p["kp"], p["vp"], p["table"].cuda(), p["lens"].cuda(),
                              max(p["lens"].tolist()) if max_len is None else max_len, p["parents"].cuda(), window_size=W, workspace=workspace, **kw)


def _check(hb, p, W=None, mask_lmk=True, expand=True, scale=None, what="", **kw):
    o, lse, ws = _call(hb, p, W, mask_lmk=mask_lmk, expand_to_chunk=expand, sm_scale=scale, **kw)
    ref = _reference(p["q"], p["k"], p["v"], p["kp"], p["vp"], p["table"], p["lens"], p["parents"], W, mask_lmk, expand,
                     scale or 1 / math.sqrt(p["q"].shape[-1]))
    _near((o, lse), ref, p["q"].dtype, what)
    return o, lse, ws


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,n,hq,hk,lens,kinds", [
    (1, 1, 1, 1, [0], ["chain"]), (1, 1, 2, 1, [1], ["star"]), (2, 1, 4, 4, [63, 64], ["chain"]),
    (4, 5, 4, 2, [65, 0, 127, 640], ["random", "star", "chain", "binary"]), (3, 9, 6, 3, [300, 1500, 129], ["random", "short", "broken"]),
    (2, 64, 2, 2, [200, 64], ["random", "chain"]), (1, 33, 8, 1, [500], ["binary"]), (2, 16, 10, 2, [70, 1], ["broken", "none"]),
    (5, 7, 3, 1, [1000, 2, 62, 0, 320], ["random", "none"]), (1, 64, 16, 1, [4000], ["binary"])])
def test_whole_cache(hb, dtype, D, B, n, hq, hk, lens, kinds):
    _check(hb, _problem(B, n, hq, hk, D, dtype, lens, kinds, seed=n))
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("W", [None, 512])
def test_many_tiles_in_one_share(hb, dtype, D, W):
    """Enough (sequence, head) pairs that the tiles are not split: a CTA walks up to 26 of them, places reused many times."""
    _check(hb, _problem(8, 3, 40, 40, D, dtype, [1600, 640, 64, 1500, 0, 321, 129, 1000], ["random", "chain"], seed=D), W)
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("W", [1, 2, 37, 64, 65, 128, 512, 100000])
@pytest.mark.parametrize("mask_lmk,expand", [(True, True), (False, False), (True, False), (False, True)])
def test_window_edges(hb, dtype, W, mask_lmk, expand):
    # lengths around the chunk borders; trees deep enough that rows of one tree see different left edges
    p = _problem(6, 20, 2, 1, 64, dtype, [0, 63, 64, 190, 701, 575], ["chain", "random"], seed=W)
    _check(hb, p, W, mask_lmk, expand, what=f"W={W}")
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_chain_over_chunk_borders_and_rows_that_see_nothing(hb, dtype):
    """Window 1 without chunks: a node sees itself only, and at a landmark position nothing."""
    p = _problem(2, 64, 2, 2, 64, dtype, [63, 100], ["chain"], seed=3)
    o, lse, _ = _check(hb, p, 1, True, False)
    pos = torch.arange(64) + torch.tensor([[63], [100]])
    assert torch.equal(torch.isneginf(lse.cpu()).all(-1), (pos + 1) % 64 == 0)
    assert not bool(o[torch.isneginf(lse)].any())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("W,expand", [(None, True), (70, False), (64, True)])
def test_nan_and_infinities_in_places_a_row_does_not_see(hb, dtype, W, expand):
    """Values and keys of one branch, of landmark places and left of the window are NaN or infinite: rows that do not see them
    are as if they were not there; rows that do are NaN."""
    B, n = 2, 12
    p = _problem(B, n, 4, 2, 64, dtype, [130, 200], ["binary"], seed=5)
    clean = {k: v.clone() for k, v in p.items()}
    o0, l0, _ = _check(hb, clean, W, True, expand)
    bad = 4                                                    # a node with children in a binary tree of 12: 9, 10
    p["v"][:, bad], p["k"][:, 7] = NAN, INF                     # 7 is a leaf
    p["v"][:, 7] = INF
    for b in range(B):                                         # landmark places of the cache, and all that lies left of the window
        T = int(p["lens"][b])
        left = 0 if W is None else ((T - W + 1) // 64 * 64 if expand else T - W + 1)
        for s in range(T):
            if s % 64 == 63 or s < left:
                pg = int(p["table"][b, s // 64])
                p["kp"][pg, :, s % 64], p["vp"][pg, :, s % 64] = NAN, NAN
    o, lse, _ = _call(hb, p, W, expand_to_chunk=expand)
    lines = _lines(p["parents"][0].tolist())
    hit = torch.tensor([bad in line or 7 in line for line in lines])
    assert torch.equal(o[:, ~hit], o0[:, ~hit]) and torch.equal(lse[:, ~hit], l0[:, ~hit])
    assert bool(torch.isnan(o[:, [bad, 9, 10, 7]]).all())
    # a NaN query spoils its own rows only
    q = {**clean, "q": clean["q"].clone()}
    q["q"][0, 3, 1] = NAN
    o, lse, _ = _call(hb, q, W, expand_to_chunk=expand)
    spoiled = torch.zeros(B, n, 4, dtype=torch.bool)
    spoiled[0, 3, 1] = True
    assert bool(torch.isnan(o[spoiled]).all()) and torch.equal(o[~spoiled], o0[~spoiled]) and bool(torch.isnan(lse[spoiled]).all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_large_scores_and_growing_maxima(hb, dtype):
    """Scores of some hundreds, and keys whose scores grow along the cache (the running maximum moves in every tile)."""
    p = _problem(1, 6, 2, 1, 64, dtype, [900], ["random"], seed=8)
    u = p["q"][0, 0, 0].float() / p["q"][0, 0, 0].float().norm()
    for c in range(15):
        pg = int(p["table"][0, c])
        rows = p["kp"][pg, 0].float()
        p["kp"][pg, 0] = (rows + u * 0.6 * c).to(dtype)
    p["q"] = (p["q"].float() * 4).to(dtype)
    _check(hb, p, None)
    _check(hb, p, 300, scale=0.5)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_one_node_is_the_decode_step_of_the_window_branch(hb, dtype):
    """A tree of one node per sequence against flex_attn_tl over the gathered cache with that token behind it."""
    hq, hk, D, W = 4, 2, 64, 128
    p = _problem(3, 1, hq, hk, D, dtype, [300, 63, 5], ["chain"], seed=2)
    o, lse, _ = _check(hb, p, W)
    for b, T in enumerate([300, 63, 5]):
        ids = p["table"][b, :(T + 63) // 64].long().cuda()
        kk, vv = (torch.cat((x[ids].transpose(1, 2).reshape(-1, hk, D)[:T], y[b])).unsqueeze(0) for x, y in ((p["kp"], p["k"]), (p["vp"], p["v"])))
        fo, fl = hb.flex_attn_tl(p["q"][b:b + 1], kk, vv, W, 64, training=False)
        tol = 2.0 ** -6 if dtype == BF else 1e-5
        assert float((fo[0].float() - o[b].float()).abs().max()) < tol and float((fl[0] - lse[b]).abs().max()) < 1e-4


def test_positions(hb):
    parents = torch.tensor([_tree("binary", 12, None), _tree("broken", 12, None), _tree("none", 12, None), _tree("chain", 12, None)], dtype=torch.int32)
    lens = torch.tensor([5, 0, 7, 1000], dtype=torch.int32)
    got = hb.draft_positions(parents.cuda(), lens.cuda()).cpu()
    want = [[int(lens[b]) + len(x) - 1 if x else -1 for x in _lines(parents[b].tolist())] for b in range(4)]
    assert got.tolist() == want
    assert hb.draft_positions(parents[:, :0].cuda(), lens.cuda()).shape == (4, 0)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_repeats_streams_workspaces_and_graphs(hb, dtype):
    p, r = (_problem(2, 12, 4, 2, 64, dtype, lens, ["random"], seed=4) for lens in ([3000, 2000], [700, 100]))
    o, lse, ws = _check(hb, p)
    again = _call(hb, p, workspace=ws)                          # the same bits, in a workspace that holds another call's
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)
    small = _call(hb, r)
    mixed = _call(hb, r, workspace=ws)
    assert torch.equal(mixed[0], small[0]) and mixed[2] is ws
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = _call(hb, p)
    s.synchronize()
    assert torch.equal(side[0], o)
    # a captured call follows lengths, tables, parents and inputs that change between replays
    args = [p["q"].clone(), p["k"].clone(), p["v"].clone(), p["kp"], p["vp"], p["table"].cuda(), p["lens"].cuda(), 3000, p["parents"].cuda()]
    hb.tree_attn_paged(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go, gl, _ = hb.tree_attn_paged(*args)
    args[6].copy_(torch.tensor([1234, 0], dtype=torch.int32))
    args[8].copy_(torch.tensor([_tree("chain", 12, None), _tree("short", 12, None)], dtype=torch.int32))
    args[0].mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    eo, el, _ = hb.tree_attn_paged(*args)
    assert torch.equal(go, eo) and torch.equal(gl, el)
    changed = {**p, "q": args[0], "lens": args[6].cpu(), "parents": args[8].cpu()}
    ref = _reference(changed["q"], p["k"], p["v"], p["kp"], p["vp"], p["table"], changed["lens"], changed["parents"], None, True, True, 0.125)
    _near((go, gl), ref, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_bad_pages_are_skipped_and_reported(hb, dtype):
    p = _problem(1, 4, 2, 2, 64, dtype, [640], ["random"], seed=6)
    for bad in (10 ** 6, -1, p["kp"].shape[0]):
        r = {**p, "table": p["table"].clone()}
        r["table"][0, 3] = bad
        o, lse, _ = _call(hb, r)
        assert _status() == 8200001
        # as if chunk 3 were not there
        keep = [c for c in range(10) if c != 3]
        t = torch.full_like(p["table"], -7)
        t[0, :9] = p["table"][0, keep]
        ref = _reference(p["q"], p["k"], p["v"], p["kp"], p["vp"], t, torch.tensor([576]), p["parents"], None, True, True, 0.125)
        _near((o, lse), ref, dtype)
    # a length past the table is cut to it, a negative one is zero
    far = {**p, "lens": torch.tensor([2 ** 31 - 1], dtype=torch.int32), "table": p["table"][:, :10].contiguous()}
    o, lse, _ = _call(hb, far, max_len=640)
    ref = _reference(p["q"], p["k"], p["v"], p["kp"], p["vp"], p["table"], p["lens"], p["parents"], None, True, True, 0.125)
    assert _status() == 8200002
    _near((o, lse), ref, dtype)
    _check(hb, {**p, "lens": torch.tensor([0], dtype=torch.int32)})
    below, zero = _call(hb, {**p, "lens": torch.tensor([-5], dtype=torch.int32)}, max_len=640), _call(hb, {**p, "lens": torch.tensor([0], dtype=torch.int32)}, max_len=640)
    assert torch.equal(below[0], zero[0]) and torch.equal(below[1], zero[1]) and _status() == 0


def test_offsets_past_32_bits(hb):
    """A pool of more than 2^32 bytes and 2^31 elements per tensor."""
    h, D, pages = 8, 128, 34000
    kp, vp = (torch.zeros(pages, h, 64, D, dtype=BF, device="cuda") for _ in range(2))
    p = _problem(2, 5, 16, h, D, BF, [150, 90], ["random"], seed=1)
    high = torch.arange(pages - 5, pages)
    for t in range(5):
        src = [(0, 0), (0, 1), (0, 2), (1, 0), (1, 1)][t]
        kp[pages - 5 + t], vp[pages - 5 + t] = p["kp"][int(p["table"][src])], p["vp"][int(p["table"][src])]
    table = p["table"].clone()
    table[0, :3], table[1, :2] = high[:3].to(torch.int32), high[3:].to(torch.int32)
    a = _call(hb, p)
    b = _call(hb, {**p, "kp": kp, "vp": vp, "table": table})
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_empty_calls(hb):
    p = _problem(2, 3, 2, 1, 64, BF, [100, 10], ["chain"])
    none = {**p, "q": p["q"][:, :0], "k": p["k"][:, :0], "v": p["v"][:, :0], "parents": p["parents"][:, :0]}
    o, lse, _ = _call(hb, {k: v.contiguous() for k, v in none.items()})
    assert o.shape == (2, 0, 2, 64) and lse.shape == (2, 0, 2)
    o, lse, _ = hb.tree_attn_paged(p["q"][:0], p["k"][:0], p["v"][:0], p["kp"], p["vp"], p["table"][:0].cuda(), p["lens"][:0].cuda(), 10,
                                   p["parents"][:0].cuda())
    assert o.shape == (0, 3, 2, 64)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,hq,hk", [(40, 3, 3), (40, 15, 3), (7, 2, 2), (64, 4, 1)])
def test_the_same_call_gives_the_same_bits(hb, dtype, D, n, hq, hk):
    """Shares of one and of many tiles, one and two row groups to a CTA: no result may hang on which warp is ahead."""
    p = _problem(8, n, hq, hk, D, dtype, [1600, 640, 64, 1500, 0, 321, 129, 1000], ["random", "chain"], seed=D)
    first = _call(hb, p)
    for _ in range(60):
        again = _call(hb, p)
        assert all(torch.equal(a, b) for a, b in zip(first[:2], again[:2]))
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,G", [(3, 200), (1, 129), (2, 1024), (64, 33)])
def test_many_heads_share_a_key_head(hb, dtype, n, G):
    """Row blocks that begin and end inside a node."""
    p = _problem(2, n, G, 1, 64, dtype, [130, 63], ["chain", "random"], seed=n + G)
    for W in (None, 100):
        _check(hb, p, W)
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
def test_two_calls_at_once(hb, dtype):
    """Calls on two streams share the SMs and their tensor memory, beside a kernel that uses it too; each has its own workspace."""
    ps = [_problem(4, 16, 8, 4, 128, dtype, [3000, 1100, 64, 700], ["random"], seed=1), _problem(3, 50, 6, 2, 64, dtype, [900, 2100, 5], ["binary"], seed=2)]
    x = [torch.randn(1, 1024, 4, 128, device="cuda").to(dtype) for _ in range(3)]
    alone = [_call(hb, p) for p in ps]
    swa = hb.flex_attn_tl(*x, window_size=256, chunk_size=64, training=False, mask_lmk=True, expand_to_chunk=True)[0]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    kept = []
    for _ in range(25):
        for p, (_, _, ws), s in zip(ps, alone, streams):
            with torch.cuda.stream(s):
                kept.append((p is ps[0], _call(hb, p, workspace=ws)))
        with torch.cuda.stream(streams[2]):
            kept.append((None, hb.flex_attn_tl(*x, window_size=256, chunk_size=64, training=False, mask_lmk=True, expand_to_chunk=True)))
    torch.cuda.synchronize()
    for first, out in kept:
        if first is None:
            assert torch.equal(out[0], swa)
        else:
            ref = alone[0 if first else 1]
            assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [100, 2000])                     # one share of the tiles, and several
def test_absent_nodes_stay_zero_beside_infinite_values(hb, dtype, D, T):
    """A value that every present row sees is infinite: those rows are not finite, absent ones are 0 and -inf all the same."""
    p = _problem(1, 6, 4, 2, D, dtype, [T], ["short"], seed=9)
    for s in (5, T - 3):
        p["vp"][int(p["table"][0, s // 64]), :, s % 64] = INF
    o, lse, _ = _call(hb, p)
    there = p["parents"][0] > -2
    assert not bool(torch.isfinite(o[0, there]).any()) and bool(torch.isfinite(lse[0, there]).all())
    assert not bool(o[0, ~there].any()) and bool(torch.isneginf(lse[0, ~there]).all())
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("W,T", [(70, 200), (600, 800)])       # one share of the tiles, and several
@pytest.mark.parametrize("expand,depth", [(False, 2), (False, 59), (False, 62), (True, 0), (True, 2)])
def test_non_finite_cache_at_the_edge_of_the_window(hb, dtype, D, W, T, expand, depth):
    """A cached token inside the window of a chain's first nodes and left of the deeper ones' (in the window's first chunk or in
    its second): rows that see it are spoiled by it, for the others it is not there."""
    p = _problem(1, 64, 4, 2, D, dtype, [T], ["chain"], seed=D + W)
    s = T - W + 1 + depth
    low = torch.tensor([(T + d - W + 1) // 64 * 64 if expand else T + d - W + 1 for d in range(64)])
    sees = low <= s
    assert s % 64 != 63 and bool(sees.any()) and not bool(sees.all())
    o0, l0, _ = _check(hb, p, W, True, expand)
    pg, at, col = int(p["table"][0, s // 64]), s % 64, D - 3
    for name, value in (("vp", INF), ("vp", NAN), ("kp", NAN)):
        r = {**p, name: p[name].clone()}
        r[name][pg, :, at] = value
        o, lse, _ = _call(hb, r, W, expand_to_chunk=expand)
        assert torch.equal(o[0, ~sees], o0[0, ~sees]) and torch.equal(lse[0, ~sees], l0[0, ~sees])
        assert not bool(torch.isfinite(o[0, sees]).any())
        assert bool(torch.isnan(lse[0, sees]).all()) if name == "kp" else torch.equal(lse, l0)
    # one element of the value: the other columns keep to the bound
    r = {**p, "vp": p["vp"].clone()}
    r["vp"][pg, :, at, col] = NAN
    o, lse, _ = _call(hb, r, W, expand_to_chunk=expand)
    assert torch.equal(o[0, ~sees], o0[0, ~sees]) and bool(torch.isnan(o[0, sees][..., col]).all())
    ref = _reference(p["q"], p["k"], p["v"], p["kp"], p["vp"], p["table"], p["lens"], p["parents"], W, True, expand, 1 / math.sqrt(D))
    o[..., col] = ref[0][..., col].to(o)
    _near((o, lse), ref, dtype)
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
def test_captured_calls_replayed_in_turn_and_at_once(hb, dtype):
    """Two captured calls of different shapes, replayed one after the other and side by side: each has a graph and scratch of its own."""
    ps = [_problem(2, 12, 4, 2, 64, dtype, [3000, 200], ["random"], seed=4), _problem(3, 9, 8, 2, 128, dtype, [900, 70, 0], ["binary"], seed=5)]
    alone, graphs, streams = [_call(hb, p) for p in ps], [], [torch.cuda.Stream() for _ in ps]
    for p in ps:
        args = [p["q"], p["k"], p["v"], p["kp"], p["vp"], p["table"].cuda(), p["lens"].cuda(), max(p["lens"].tolist()), p["parents"].cuda()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = hb.tree_attn_paged(*args)
        graphs.append((graph, out, args))
    for side_by_side in (False, True):
        for _ in range(10):
            for graph, out, _ in graphs:
                out[0].fill_(NAN), out[1].fill_(NAN)
            torch.cuda.synchronize()
            for (graph, _, _), s in zip(graphs, streams if side_by_side else [torch.cuda.current_stream()] * 2):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for (_, out, _), ref in zip(graphs, alone):
                assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    assert _status() == 0
