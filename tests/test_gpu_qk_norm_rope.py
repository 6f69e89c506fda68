"""Norm and rotation of queries and keys against the formulas in 64 bits, forward and backward.  Needs a B200.

Tolerances.  The kernel computes in fp32 and rounds once.  An output is a sum of two products of |a|, |b| <= m (the largest
entry of the row) with cos and sin; each factor carries at most 8 roundings of 2^-24 and the angle 4e-7, so the fp32 part is
within 3e-6 m of the exact value, and the final rounding adds half a step of the output's type relative to the value.  dx adds
a mean over the row of the same quality: 6e-6 m.  dw is a sum over N rows in fp32: at most 64 additions in a chain and a tree
behind them here, 1e-5 of the sum of the terms' magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def hb():
    import hils_attention_b200 as pkg
    return pkg


def _pairs(rot, interleaved):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def _turn(x, pos, inv_freq, interleaved, scaling, sign=1.0):
    a, b = _pairs(2 * inv_freq.numel(), interleaved)
    t = sign * pos.double()[..., None] * inv_freq.double()
    c, s = torch.cos(t)[:, :, None] * scaling, torch.sin(t)[:, :, None] * scaling
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def _formula(x, w, pos, inv_freq, eps, interleaved, scaling, g):
    """(out, dx, dw, magnitude of dw's terms) in 64 bits on the CPU."""
    x, g = x.detach().double().cpu(), g.double().cpu()
    pos = pos.cpu().expand(x.shape[0], x.shape[1])
    inv_freq = inv_freq.cpu()
    w = None if w is None else w.detach().double().cpu()
    r = torch.ones(()) if w is None else 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    out = _turn(x * r * (1 if w is None else w), pos, inv_freq, interleaved, scaling)
    dy = _turn(g, pos, inv_freq, interleaved, scaling, -1.0)
    if w is None:
        return out, dy, None, None
    n = x * r
    dx = r * (w * dy - n * (w * dy * n).mean(-1, keepdim=True))
    return out, dx, (dy * n).sum((0, 1, 2)), (dy * n).abs().sum((0, 1, 2))


def _near(x, ref, c, what):
    assert x.shape == ref.shape
    step = 0.5 * torch.finfo(x.dtype).eps
    got = x.detach().double().cpu()
    m = ref.abs().amax(-1, keepdim=True) if ref.numel() else ref
    bad = (got - ref).abs() > step * ref.abs() + c * m
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - ref).abs().max()):.3e}"


def _check(hb, q, k, pos, inv_freq, qw, kw, interleaved=False, scaling=1.0, eps=1e-6, seed=0):
    leaves = [t.requires_grad_(True) if t is not None and t.is_leaf else t for t in (q, k, qw, kw)]
    outs = hb.qk_norm_rope(q, k, pos, inv_freq, qw, kw, eps=eps, interleaved=interleaved, attention_scaling=scaling)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    gs = [None if o is None else torch.randn(o.shape, device="cuda", generator=gen).to(o.dtype) for o in outs]
    wanted = [t for t in leaves if t is not None]
    got = dict(zip(map(id, wanted), torch.autograd.grad([o for o in outs if o is not None], wanted, [g for g in gs if g is not None])))
    for name, x, w, o, g in (("q", q, qw, outs[0], gs[0]), ("k", k, kw, outs[1], gs[1])):
        if x is None:
            assert o is None
            continue
        out, dx, dw, mag = _formula(x, w, pos, inv_freq, eps, interleaved, scaling, g)
        assert o.dtype == x.dtype and o.is_contiguous()
        _near(o, out, 3e-6, name)
        _near(got[id(x)], dx, 6e-6, "d" + name)
        if w is not None:
            d = got[id(w)]
            bad = (d.double().cpu() - dw).abs() > 0.5 * torch.finfo(d.dtype).eps * dw.abs() + 1e-5 * mag
            assert not bool(bad.any()), f"d{name}_weight"
    return outs


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("B,L,hq,hk,D,rot,dtype", [
    (1, 1, 1, 1, 64, 64, BF), (2, 7, 4, 2, 128, 128, BF), (3, 1, 32, 8, 128, 64, BF), (1, 33, 5, 1, 80, 40, BF), (2, 9, 3, 3, 256, 256, BF),
    (1, 5, 2, 2, 34, 10, BF), (2, 3, 2, 1, 2, 2, BF), (1, 4, 2, 2, 96, 0, BF), (2, 65, 6, 2, 96, 48, F32), (1, 3, 2, 2, 250, 250, F32),
    (1, 300, 17, 1, 64, 64, F32), (2, 6, 4, 4, 256, 128, F32), (1, 1000, 16, 16, 64, 64, BF), (1, 2, 1, 1, 192, 192, BF)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_against_the_formulas(hb, B, L, hq, hk, D, rot, dtype, interleaved):
    q, k = _rand((B, L, hq, D), dtype, 1), _rand((B, L, hk, D), dtype, 2)
    qw, kw = 1 + 0.2 * _rand((D,), dtype, 3), 1 + 0.2 * _rand((D,), dtype, 4)
    pos = torch.randint(0, 100000, (B, L), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    f, s = hb.rope_frequencies(rot, device="cuda")
    _check(hb, q, k, pos, f, qw, kw, interleaved, 1.25)


def test_without_norms_with_one_norm_and_without_keys(hb):
    B, L, D = 2, 11, 64
    f = hb.rope_frequencies(D, device="cuda")[0]
    pos = torch.arange(L, device="cuda", dtype=torch.int32)
    mk = lambda: (_rand((B, L, 4, D), BF, 1), _rand((B, L, 2, D), BF, 2))
    w = lambda: 1 + 0.2 * _rand((D,), BF, 3)
    _check(hb, *mk(), pos, f, None, None)
    _check(hb, *mk(), pos, f, w(), None)
    _check(hb, *mk(), pos[None], f, None, w())
    _check(hb, mk()[0], None, pos, f, w(), None)
    # fp32 weights of a bf16 model keep their bits
    _check(hb, *mk(), pos, f, w().float() + 1e-4, w().float() + 1e-4)


@pytest.mark.parametrize("dtype,interleaved", [(F32, False), (F32, True), (BF, False)])
def test_far_and_negative_positions_keep_their_angles(hb, dtype, interleaved):
    D = 64
    pos = torch.tensor([[0, 1, -1, 1000003, 2 ** 31 - 1, -(2 ** 31), 16777217]], device="cuda")
    f, s = hb.rope_frequencies(D, scaling="yarn", factor=16.0, device="cuda")
    for p in (pos, pos.to(torch.int32)):
        # the reference's own angle: at 2^31 the fp64 product of position and frequency is good to 2^31 * 2^-53 rad
        _check(hb, _rand((1, 7, 2, D), dtype, 1), _rand((1, 7, 1, D), dtype, 2), p, f, None, None, interleaved, s)
    far = torch.full((1, 7), 10 ** 9, device="cuda")
    _check(hb, _rand((1, 7, 2, D), dtype, 1), _rand((1, 7, 1, D), dtype, 2), far, f.float(), None, None, interleaved, s)


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
def test_slices_of_a_fused_projection_and_odd_strides(hb, offset):
    B, L, hq, hk, D = 2, 9, 4, 2, 64
    buf = _rand((B, L, (hq + 2 * hk) * D + offset), BF, 7)
    x = buf[..., offset:]
    q, k = x[..., :hq * D].unflatten(-1, (hq, D)).detach(), x[..., hq * D:(hq + hk) * D].unflatten(-1, (hk, D)).detach()
    f = hb.rope_frequencies(D, device="cuda")[0]
    pos = torch.randint(0, 5000, (B, L), device="cuda")
    qw, kw = 1 + 0.2 * _rand((D,), BF, 3), 1 + 0.2 * _rand((D,), BF, 4)
    _check(hb, q, k, pos, f, qw, kw)
    # token-major, transposed heads, an expanded batch, a last dimension with a stride
    t = _rand((B, hq, L, D), BF, 8).transpose(1, 2).detach()
    e = _rand((1, L, hk, D), BF, 9).expand(B, L, hk, D).detach()
    _check(hb, t, e, pos, f, qw.detach(), kw.detach())
    s = _rand((B, L, hq, 2 * D), BF, 10)[..., ::2].detach()
    _check(hb, s, e, pos, f, qw.detach(), kw.detach())


def test_gradients_of_broadcast_inputs_and_outputs(hb):
    """Keys shared by a batch, and a loss whose gradient is one number spread over the output."""
    B, L, D = 3, 5, 64
    f = hb.rope_frequencies(D, device="cuda")[0]
    pos = torch.randint(0, 3000, (B, L), device="cuda")
    k0 = _rand((1, L, 2, D), F32, 1).requires_grad_(True)
    w = (1 + 0.2 * _rand((D,), F32, 2)).requires_grad_(True)
    q = _rand((B, L, 2, D), F32, 3)
    _, ko = hb.qk_norm_rope(q, k0.expand(B, L, 2, D), pos, f, None, w)
    ko.sum().backward()
    _, dx, dw, mag = _formula(k0.expand(B, L, 2, D), w, pos, f, 1e-6, False, 1.0, torch.ones(B, L, 2, D))
    dx = dx.sum(0, keepdim=True)
    assert float((k0.grad.double().cpu() - dx).abs().max()) <= 3 * 6e-6 * float(dx.abs().max() + 1)
    assert bool(((w.grad.double().cpu() - dw).abs() <= 2.0 ** -24 * dw.abs() + 1e-5 * mag).all())


def test_gradients_against_differences(hb):
    """Central differences of the fp32 forward.  f(x +- h) of outputs of size ~2 carries 2^-23 each; with h = 2^-6 the sum
    over D = 64 outputs of a row is off by 64 * 2^-22 / 2^-5 < 5e-4, the third-derivative term h^2/6 * f''' by a few 1e-4."""
    D = 64
    f = hb.rope_frequencies(32, device="cuda")[0]
    pos = torch.tensor([[3, 70, 1234]], device="cuda")
    q, w, g = _rand((1, 3, 2, D), F32, 1), 1 + 0.2 * _rand((D,), F32, 2), _rand((1, 3, 2, D), F32, 3)
    q.requires_grad_(True), w.requires_grad_(True)
    o, _ = hb.qk_norm_rope(q, None, pos, f, w, interleaved=True)
    dq, dw = torch.autograd.grad(o, (q, w), g)
    h = 2.0 ** -6

    def value(x, u):
        return (hb.qk_norm_rope(x, None, pos, f, u, interleaved=True)[0].double() * g.double()).sum().item()
    with torch.no_grad():
        for at in ((0, 0, 0, 0), (0, 1, 1, 17), (0, 2, 0, 31), (0, 2, 1, 63)):
            e = torch.zeros_like(q)
            e[at] = h
            assert abs((value(q + e, w) - value(q - e, w)) / (2 * h) - float(dq[at])) < 4e-3
        for d in (0, 1, 33):
            e = torch.zeros_like(w)
            e[d] = h
            assert abs((value(q, w + e) - value(q, w - e)) / (2 * h) - float(dw[d])) < 4e-3


def test_only_what_needs_a_gradient_gets_one_and_empty_calls(hb):
    D = 64
    f = hb.rope_frequencies(D, device="cuda")[0]
    pos = torch.arange(4, device="cuda")
    q, k, w = _rand((1, 4, 2, D), BF, 1), _rand((1, 4, 1, D), BF, 2).requires_grad_(True), _rand((D,), BF, 3).requires_grad_(True)
    qo, ko = hb.qk_norm_rope(q, k, pos, f, w, None)
    (ko.float().sum() + 2 * qo.float().sum()).backward()
    assert q.grad is None and k.grad is not None and w.grad is not None
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(hb.qk_norm_rope(k, None, pos, f)[0].float().square().sum(), k, create_graph=True)[0].sum(), k)
    for B, L, hq in ((0, 4, 2), (1, 0, 2), (1, 4, 0)):
        x, kk = torch.empty(B, L, hq, D, device="cuda", dtype=BF).requires_grad_(True), _rand((B, L, 1, D), BF, 2).requires_grad_(True)
        u = torch.ones(D, device="cuda", dtype=BF, requires_grad=True)
        a, b = hb.qk_norm_rope(x, kk, torch.arange(L, device="cuda"), f, u, u)
        (a.float().sum() + b.float().sum()).backward()
        assert a.shape == x.shape and x.grad.shape == x.shape and bool(torch.isfinite(u.grad).all())


def test_large_offsets_repeat_and_stream(hb):
    """More than 2^31 elements in one tensor; the same call gives the same bits, weight gradients included."""
    D, H, L = 128, 32, 540000                                  # 2.2e9 elements
    q = torch.zeros(1, L, H, D, dtype=BF, device="cuda")
    q[0, -1] = _rand((H, D), BF, 1)
    f = hb.rope_frequencies(D, device="cuda")[0]
    w = 1 + 0.2 * _rand((D,), BF, 2)
    pos = torch.arange(L, device="cuda", dtype=torch.int32)
    o, _ = hb.qk_norm_rope(q, None, pos, f, w)
    ref = _formula(q[:, -1:], w, pos[-1:], f, 1e-6, False, 1.0, torch.zeros(1, 1, H, D))[0]
    _near(o[:, -1:], ref, 3e-6, "last token")
    assert not bool(o[0, :1000].any())
    del q, o
    x, k, g = _rand((1, 3000, 8, D), BF, 3).requires_grad_(True), _rand((1, 3000, 4, D), BF, 4).requires_grad_(True), _rand((1, 3000, 8, D), BF, 5)
    u = w.clone().requires_grad_(True)

    def once():
        a, b = hb.qk_norm_rope(x, k, pos[:3000], f, u, u)
        return [a, b, *torch.autograd.grad((a, b), (x, k, u), (g, g[:, :, :4]))]
    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_forward_and_backward_in_a_graph(hb):
    """Forward and backward of fresh leaves captured together; replays follow the inputs."""
    D = 64
    f = hb.rope_frequencies(D, device="cuda")[0]
    q, g, w = _rand((2, 6, 4, D), BF, 1), _rand((2, 6, 4, D), BF, 2), 1 + 0.2 * _rand((D,), BF, 3)
    pos = torch.arange(6, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        x, u = q.detach().requires_grad_(True), w.detach().requires_grad_(True)
        o, _ = hb.qk_norm_rope(x, None, pos, f, u)
        return [o.detach(), *torch.autograd.grad(o, (x, u), g)]
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    q.copy_(_rand((2, 6, 4, D), BF, 11))
    pos.add_(900)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in outs]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_one_rounding_against_the_table_form(hb):
    """rmsnorm_rope with a table at the same positions: it rounds three times (after the norm, the weight and the rotation,
    as the reference does), so the two agree within 2.5 steps of the largest entry of a pair."""
    B, L, H, D = 2, 40, 3, 128
    x, w = _rand((B, L, H, D), BF, 1), 1 + 0.2 * _rand((D,), BF, 2)
    f = hb.rope_frequencies(D, device="cuda")[0]
    pos = torch.randint(0, 4000, (B, L), device="cuda")
    t = (pos.double()[..., None] * f).repeat(1, 1, 2)
    old = hb.rmsnorm_rope(x, w, torch.cos(t).float(), torch.sin(t).float())
    new, _ = hb.qk_norm_rope(x, None, pos, f, w)
    a, b = new.float().unflatten(-1, (2, D // 2)), old.float().unflatten(-1, (2, D // 2))
    size = a.square().sum(-2, keepdim=True).sqrt()
    assert bool(((a - b).abs() <= 2.5 * 2.0 ** -7 * size + 1e-6).all())


def test_forward_mode_is_refused(hb):
    """No forward-mode formula is offered: a tangent is refused, not dropped, whether or not gradients are recorded."""
    import torch.autograd.forward_ad as fw
    q, k, w = torch.randn(1, 3, 2, 64, device="cuda"), torch.randn(1, 3, 1, 64, device="cuda"), torch.ones(64, device="cuda")
    pos, freq = torch.arange(3, device="cuda"), hb.rope_frequencies(64, device="cuda")[0]
    plain = hb.qk_norm_rope(q, k, pos, freq, w, w)
    with fw.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(hb.qk_norm_rope(q, k, pos, freq, w, w), plain))     # no tangent among them
        for i, x in enumerate((q, k, w, w)):
            args = [q, k, w, w]
            args[i] = fw.make_dual(x, torch.ones_like(x))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                    hb.qk_norm_rope(args[0], args[1], pos, freq, args[2], args[3])
