"""Workloads of the position, drafted-tree and page operators: inputs, plain forms and values in 64 bits.

Four operators: `rope` (norm of queries and keys per head with the rotation of their positions), `tree` (attention of a
tree of drafted tokens over the paged store), `copy` (pages of the store copied for a fork or a compaction) and `commit`
(the accepted path of a drafted tree written into the pages).  `run` is one pass; with `own` set it goes through the
framework's entry points, otherwise through elementary torch operations in 32 bits.
"""
import math

import torch

own = False

PAGE = 64            # tokens of a page, and of a chunk


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _rope(**kw):
    case = {"op": "rope", "dtype": "bf16", "B": 1, "L": 1, "h_q": 4, "h_k": 4, "D": 64, "rot": 64, "interleaved": False, "norm": True,
            "fused": False, "far": 4096, "factor": 1.0, "train": False}
    return {**case, **kw}


def _tree(**kw):
    case = {"op": "tree", "dtype": "bf16", "B": 1, "n": 8, "h_q": 4, "h_kv": 2, "D": 64, "window": 512, "short": 600, "long": 700, "ragged": False}
    return {**case, **kw}


def _copy(**kw):
    case = {"op": "copy", "dtype": "bf16", "layers": 1, "pairs": 1, "h_kv": 2, "D": 64}
    return {**case, **kw}


def _commit(**kw):
    case = {"op": "commit", "dtype": "bf16", "layers": 1, "B": 1, "n": 8, "h_kv": 2, "D": 64}
    return {**case, **kw}


def listed():
    return [
        # one new token of each of 8 sequences at positions of their own: latency
        {"name": "rope_decode", **_rope(B=8, L=1, h_q=32, h_k=8, D=128, rot=128, far=131072)},
        # a training step's batch of 8192 tokens, 16 heads of 64
        {"name": "rope_train_8k", **_rope(B=1, L=8192, h_q=16, h_k=16, D=64, rot=64, train=True)},
        # the 64K-token context with 32 heads of 128, queries and keys as slices of one projection
        {"name": "rope_train_64k", **_rope(B=1, L=65536, h_q=32, h_k=32, D=128, rot=128, fused=True, train=True)},
        # half of an odd-sized head rotated, interleaved pairs, fp32, stretched frequencies
        {"name": "rope_partial_f32", **_rope(dtype="f32", B=3, L=1021, h_q=6, h_k=2, D=96, rot=48, interleaved=True, norm=False,
                                            far=200000, factor=8.0, train=True)},
        # five drafted tokens of one sequence, a short window: latency
        {"name": "tree_small", **_tree(B=1, n=5, h_q=4, h_kv=2, D=64, window=128, short=640, long=640)},
        # the window branch of a drafted step of 32 sequences, 32 heads of 128, trees of up to 16 nodes
        {"name": "tree_window_b32", **_tree(B=32, n=16, h_q=32, h_kv=32, D=128, window=512, short=1100, long=4000, ragged=True)},
        # the whole cache of long sequences, four query heads for each key head, the widest tree
        {"name": "tree_whole_32k", **_tree(B=4, n=64, h_q=32, h_kv=8, D=128, window=0, short=32000, long=32700)},
        # fp32, odd sizes
        {"name": "tree_f32", **_tree(dtype="f32", B=2, n=9, h_q=6, h_kv=3, D=64, window=0, short=1501, long=2003, ragged=True)},
        # the last page of a sequence copied for a second continuation
        {"name": "copy_fork", **_copy(layers=2, pairs=1, h_kv=2, D=64)},
        # half of a pool moved, four layers
        {"name": "copy_many", **_copy(layers=4, pairs=512, h_kv=8, D=128)},
        # one sequence's accepted path, one layer
        {"name": "commit_small", **_commit(layers=1, B=1, n=8, h_kv=2, D=64)},
        # 32 sequences, 16 layers
        {"name": "commit_b32", **_commit(layers=16, B=32, n=16, h_kv=8, D=128)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "tree", "tree", "tree", "copy", "commit"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "rope":
        D = rng.choice([64, 80, 96, 128, 192])
        h_k = rng.choice([1, 2, 3, 4, 8, 16])
        h_q = h_k * rng.choice([1, 2, 3, 4])
        B, L = rng.choice([(rng.randint(1, 48), 1), (rng.randint(1, 6), _log(rng, 2, 4000))])
        return _rope(dtype=dtype, B=B, L=L, h_q=h_q, h_k=h_k, D=D, rot=rng.choice([D, D, D // 2]), interleaved=rng.random() < 0.4,
                     norm=rng.random() < 0.7, fused=rng.random() < 0.4, far=_log(rng, 4096, 1000000), factor=rng.choice([1.0, 4.0, 16.0]),
                     train=rng.random() < 0.6)
    if op == "tree":
        D = rng.choice([64, 128])
        h_kv = rng.choice([1, 2, 4, 5, 8])
        h_q = h_kv * rng.choice([1, 2, 3, 4, 8])
        window = rng.choice([0, 0, 128, 512, 777])
        long = _log(rng, 1, 20000 if dtype == "bf16" else 6000)
        return _tree(dtype=dtype, B=rng.randint(1, 4 if dtype == "bf16" else 3), n=rng.randint(1, 64 if dtype == "bf16" else 24), h_q=h_q,
                     h_kv=h_kv, D=D, window=window, short=max(0, int(long * rng.uniform(0.3, 1.0))), long=long, ragged=rng.random() < 0.5)
    if op == "copy":
        return _copy(dtype=dtype, layers=rng.randint(1, 4), pairs=_log(rng, 1, 300), h_kv=rng.randint(1, 6), D=rng.choice([64, 128]))
    return _commit(dtype=dtype, layers=rng.randint(1, 12), B=rng.randint(1, 24), n=rng.randint(1, 48), h_kv=rng.randint(1, 6),
                   D=rng.choice([64, 128]))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _lengths(case, g):
    return torch.randint(case["short"], case["long"] + 1, (case["B"],), generator=g, device="cuda", dtype=torch.int32)


def _parents(B, n, ragged, g):
    """Trees of drafted tokens: a node's parent is one of the few nodes before it, or the last cached token (-1); in a
    ragged batch a sequence's last places may be empty (-2)."""
    j = torch.arange(n, device="cuda")
    back = torch.randint(1, 5, (B, n), generator=g, device="cuda")
    parents = (j - back).clamp_min(-1)
    if ragged:
        used = torch.randint((n + 1) // 2, n + 1, (B, 1), generator=g, device="cuda")
        parents = torch.where(j < used, parents, -2)
    return parents.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    T = _type(case)

    def rand(*shape, dtype=T, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    if case["op"] == "rope":
        B, L, h_q, h_k, D, rot = (case[k] for k in ("B", "L", "h_q", "h_k", "D", "rot"))
        if case["fused"]:        # slices of one projection
            qkv = rand(B, L, h_q + 2 * h_k, D)
            q, k = qkv[:, :, :h_q], qkv[:, :, h_q:h_q + h_k]
        else:
            q, k = rand(B, L, h_q, D), rand(B, L, h_k, D)
        start = torch.randint(0, max(1, case["far"] - L), (B, 1), generator=g, device="cuda")
        positions = start + torch.arange(L, device="cuda")
        inv_freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot) / case["factor"]
        s = {"q": q, "k": k, "positions": positions, "inv_freq": inv_freq, "q_weight": None, "k_weight": None,
             "interleaved": case["interleaved"], "scaling": 0.1 * math.log(case["factor"]) + 1.0, "train": case["train"], "op": "rope"}
        if case["norm"]:
            s["q_weight"], s["k_weight"] = 1.0 + 0.1 * rand(D), 1.0 + 0.1 * rand(D)
        if case["train"]:
            s["d_q"], s["d_k"] = rand(B, L, h_q, D), rand(B, L, h_k, D)
            for name in ("q", "k", "q_weight", "k_weight"):
                if s[name] is not None:
                    s[name].requires_grad_(True) if s[name].is_leaf else None
                    s[name] = s[name] if s[name].requires_grad else s[name].detach().requires_grad_(True)
        return s
    if case["op"] == "tree":
        B, n, h_q, h_kv, D = (case[k] for k in ("B", "n", "h_q", "h_kv", "D"))
        width = (case["long"] + n) // PAGE + 1
        pool = B * width + 1
        order = torch.randperm(pool - 1, generator=g, device="cuda") + 1           # page 0 is nobody's
        s = {"q": rand(B, n, h_q, D), "k": rand(B, n, h_kv, D), "v": rand(B, n, h_kv, D), "k_pages": rand(pool, h_kv, PAGE, D),
             "v_pages": rand(pool, h_kv, PAGE, D), "table": order[:B * width].view(B, width).to(torch.int32).contiguous(),
             "lens": _lengths(case, g), "max_len": case["long"], "parents": _parents(B, n, case["ragged"], g),
             "window": case["window"] or None, "op": "tree"}
        return s
    if case["op"] == "copy":
        layers, pairs, h_kv, D = (case[k] for k in ("layers", "pairs", "h_kv", "D"))
        pool = 2 * pairs + 1
        order = (torch.randperm(pool - 1, generator=g, device="cuda") + 1).cpu().to(torch.int32)
        src, dst = order[:pairs].contiguous(), order[pairs:].contiguous()          # what the host keeps of a pool's pages
        return {"k_pages": rand(layers, pool, h_kv, PAGE, D), "v_pages": rand(layers, pool, h_kv, PAGE, D), "src": src, "dst": dst,
                "src_index": src.long().cuda(), "dst_index": dst.long().cuda(), "op": "copy"}
    layers, B, n, h_kv, D = (case[k] for k in ("layers", "B", "n", "h_kv", "D"))
    lens = torch.randint(0, 200, (B,), generator=g, device="cuda", dtype=torch.int32)
    width = (200 + n) // PAGE + 1
    pool = B * width + 1
    order = torch.randperm(pool - 1, generator=g, device="cuda") + 1
    # the accepted path: ascending node ids, then -1; between none and all of the nodes
    took = torch.randint(0, n + 1, (B, 1), generator=g, device="cuda")
    nodes = torch.rand(B, n, generator=g, device="cuda").argsort(1)
    nodes = torch.where(torch.arange(n, device="cuda") < took, nodes, n).sort(1).values
    path = torch.where(nodes < n, nodes, -1).to(torch.int32)
    return {"k": rand(layers, B, n, h_kv, D), "v": rand(layers, B, n, h_kv, D), "k_pages": rand(layers, pool, h_kv, PAGE, D),
            "v_pages": rand(layers, pool, h_kv, PAGE, D), "table": order[:B * width].view(B, width).to(torch.int32).contiguous(),
            "lens": lens, "path": path, "op": "commit"}


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _plain_rotate(x, weight, cos, sin, rot, interleaved):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    turned, rest = y[..., :rot], y[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _plain_rope(s):
    angle = s["positions"].double().unsqueeze(-1) * s["inv_freq"]                  # in 64 bits: positions reach a million
    cos, sin = ((f(angle) * s["scaling"]).float().unsqueeze(2) for f in (torch.cos, torch.sin))
    rot = 2 * s["inv_freq"].numel()
    return tuple(_plain_rotate(x, w, cos, sin, rot, s["interleaved"]) for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _plain_tree(s):
    q, table, lens, parents, W = s["q"], s["table"].long(), s["lens"].long(), s["parents"].long(), s["window"]
    B, n, h_q, D = q.shape
    h_kv = s["k"].shape[2]
    # the pages that some row may see: all of them, or those from the chunk of the first row's left edge on
    chunks = table.shape[1] if W is None else min(table.shape[1], (W + PAGE - 2) // PAGE + 2)
    first = torch.zeros_like(lens) if W is None else ((lens - W + 1).clamp_min(0) // PAGE).clamp_max(table.shape[1] - chunks)
    c = first[:, None] + torch.arange(chunks, device=q.device)
    token = (c[:, :, None] * PAGE + torch.arange(PAGE, device=q.device)).flatten(1)                      # (B, m)
    pages = table.gather(1, c)
    held = token < lens[:, None]
    k, v = (x[pages].float().transpose(2, 3).flatten(1, 2) for x in (s["k_pages"], s["v_pages"]))      # (B, m, h_kv, D)
    k, v = (torch.where(held[..., None, None], x, 0.0) for x in (k, v))
    k, v = torch.cat((k, s["k"].float()), 1), torch.cat((v, s["v"].float()), 1)
    # ancestors: row j of (I + A)^n is non-zero at j's ancestors and itself
    there = parents > -2
    step = torch.eye(n, device=q.device) + (parents.clamp_min(-1)[..., None] == torch.arange(n, device=q.device))
    line = (torch.matrix_power(step, n) > 0) & there[..., None] & there[:, None, :]
    at = lens[:, None] + line.sum(-1) - 1                                                               # (B, n) positions
    low = torch.full_like(at, -1 << 40) if W is None else torch.div(at - W + 1, PAGE, rounding_mode="floor") * PAGE
    key_at = torch.cat((token, at), 1)
    sees = torch.cat((held[:, None, :].expand(B, n, -1), line), 2)
    sees = sees & (key_at[:, None, :] >= low[..., None]) & ((key_at + 1) % PAGE != 0)[:, None, :] & there[..., None]
    scores = torch.einsum("bnhgd,bmhd->bhgnm", q.float().view(B, n, h_kv, h_q // h_kv, D), k) / math.sqrt(D)
    scores = scores.masked_fill(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top.clamp_min(-3e38))
    total = e.sum(-1, keepdim=True)
    o = torch.einsum("bhgnm,bmhd->bnhgd", e / total.clamp_min(1e-30), v).reshape(B, n, h_q, D)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(B, n, h_q)
    return o.to(q.dtype), lse


def _plain_copy(s):
    s["k_pages"][:, s["dst_index"]] = s["k_pages"][:, s["src_index"]]
    s["v_pages"][:, s["dst_index"]] = s["v_pages"][:, s["src_index"]]
    return s["k_pages"], s["v_pages"]


def _plain_commit(s):
    path = s["path"].long()
    b, i = (path >= 0).nonzero(as_tuple=True)
    node, token = path[b, i], s["lens"].long()[b] + i
    page, row = s["table"].long()[b, token // PAGE], token % PAGE
    s["k_pages"][:, page, :, row] = s["k"][:, b, node].transpose(0, 1)
    s["v_pages"][:, page, :, row] = s["v"][:, b, node].transpose(0, 1)
    return s["k_pages"], s["v_pages"]


def run(state):
    s = state
    if own:
        import hils_attention_b200 as hb
    if s["op"] == "rope":
        if own:
            outs = hb.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                                   interleaved=s["interleaved"], attention_scaling=s["scaling"])
        else:
            outs = _plain_rope(s)
        if not s["train"]:
            return outs
        leaves = [x for x in (s["q"], s["k"], s["q_weight"], s["k_weight"]) if x is not None]
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, (s["d_q"], s["d_k"])))
    if s["op"] == "tree":
        if not own:
            return _plain_tree(s)
        o, lse, s["workspace"] = hb.tree_attn_paged(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["max_len"],
                                                    s["parents"], window_size=s["window"], workspace=s.get("workspace"))
        return o, lse
    if s["op"] == "copy":
        if not own:
            return _plain_copy(s)
        hb.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
        return s["k_pages"], s["v_pages"]
    if not own:
        return _plain_commit(s)
    hb.commit_drafts(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["path"])
    return s["k_pages"], s["v_pages"]


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rope":
        elements = case["B"] * case["L"] * (case["h_q"] + case["h_k"]) * case["D"]
        return {"bytes": elements * size * (4 if case["train"] else 2) + case["B"] * case["L"] * 8, "flops": elements * (24 if case["train"] else 9)}
    if case["op"] == "tree":
        B, n, h_q, h_kv, D = (case[k] for k in ("B", "n", "h_q", "h_kv", "D"))
        seen = (case["short"] + case["long"]) / 2
        if case["window"]:
            seen = min(seen, case["window"] + PAGE / 2)
        return {"bytes": B * (seen * h_kv * D * 2 + 2 * n * h_kv * D + 2 * n * h_q * D) * size + B * n * h_q * 4,
                "flops": B * n * h_q * (seen + n / 4) * 4 * D}
    if case["op"] == "copy":
        return {"bytes": case["layers"] * case["pairs"] * case["h_kv"] * PAGE * case["D"] * size * 2 * 2, "flops": 0}
    return {"bytes": case["layers"] * case["B"] * (case["n"] / 2) * case["h_kv"] * case["D"] * size * 2 * 2 + case["B"] * case["n"] * 4, "flops": 0}


# ---------------------------------------------------------------------------------------------------------------
# values in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------
def _exact_rope(s):
    rot, D = 2 * s["inv_freq"].numel(), s["q"].shape[-1]
    turn = torch.polar(torch.full_like(s["inv_freq"], s["scaling"]).expand(*s["positions"].shape, -1).contiguous(),
                       s["positions"].double()[..., None] * s["inv_freq"])[:, :, None]                # (B, L, 1, rot/2) complex
    low = torch.arange(0, rot, 2) if s["interleaved"] else torch.arange(rot // 2)
    high = low + (1 if s["interleaved"] else rot // 2)

    def rotated(x, by):
        y = x.clone()
        z = torch.complex(x[..., low], x[..., high]) * by
        y[..., low], y[..., high] = z.real, z.imag
        return y

    outs, grads, of_weights = [], [], []
    for name in ("q", "k"):
        x, w = s[name].detach().double(), s[name + "_weight"]
        w = None if w is None else w.detach().double()
        r = 1.0 if w is None else (x.square().sum(-1, keepdim=True) / D + 1e-6) ** -0.5
        outs.append(rotated(x * r * (1.0 if w is None else w), turn))
        if s["train"]:
            back = rotated(s["d_" + name].double(), turn.conj())
            if w is None:
                grads.append(back)
            else:
                unit = x * r
                of_weights.append((back * unit).sum((0, 1, 2)))
                back = back * w
                grads.append(r * (back - unit * (back * unit).sum(-1, keepdim=True) / D))
    return tuple(outs + grads + of_weights)


def _exact_tree(s):
    B, n, h_q, D = s["q"].shape
    h_kv = s["k"].shape[2]
    outs, sums = [], []
    for b in range(B):
        length, parents = int(s["lens"][b]), s["parents"][b].tolist()
        held = -(-length // PAGE)
        pages = s["table"][b, :held].long()
        k, v = (x[pages].double().permute(1, 0, 2, 3).reshape(h_kv, held * PAGE, D)[:, :length] for x in (s["k_pages"], s["v_pages"]))
        k, v = (torch.cat((x, y[b].double().transpose(0, 1)), 1) for x, y in ((k, s["k"]), (v, s["v"])))     # (h_kv, length + n, D)
        lines = []
        for j in range(n):
            lines.append([] if parents[j] < -1 else ([j] if parents[j] < 0 else lines[parents[j]] + [j]))
        at = torch.arange(length + n)
        sees = torch.zeros(n, length + n, dtype=torch.bool)
        for j, line in enumerate(lines):
            at[length + j] = length + len(line) - 1
        for j, line in enumerate(lines):
            if line:
                sees[j, :length] = True
                sees[j, [length + i for i in line]] = True
                if s["window"]:
                    sees[j] &= at >= (int(at[length + j]) - s["window"] + 1) // PAGE * PAGE
        sees &= (at + 1) % PAGE != 0
        score = torch.matmul(s["q"][b].double().view(n, h_kv, -1, D).permute(1, 2, 0, 3), k[:, None].transpose(-1, -2)) * D ** -0.5
        score = score.masked_fill(~sees.cuda(), -math.inf)
        total = torch.logsumexp(score, -1)
        p = torch.where(torch.isinf(total)[..., None], 0.0, torch.exp(score - total[..., None]))
        outs.append(torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).reshape(n, h_q, D))
        sums.append(total.permute(2, 0, 1).reshape(n, h_q))
    return torch.stack(outs), torch.stack(sums)


def _exact_pages(s):
    new = [s["k_pages"].double(), s["v_pages"].double()]
    old = [s["k_pages"], s["v_pages"]]
    if s["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for x, y in zip(new, old):
                x[:, b] = y[:, a].double()
        return tuple(new)
    for b, nodes in enumerate(s["path"].tolist()):
        for i, node in enumerate(x for x in nodes if x >= 0):
            token = int(s["lens"][b]) + i
            page = int(s["table"][b, token // PAGE])
            for x, y in zip(new, (s["k"], s["v"])):
                x[:, page, :, token % PAGE] = y[:, b, node].double()
    return tuple(new)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "copy": _exact_pages, "commit": _exact_pages}[case["op"]](s)
