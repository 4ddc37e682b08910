"""Rotary positions with several axes and the query / key norms with the rotation in the same pass
(fp4t_rotary, fp4t_qk_norm_rotary_forward / _backward) against the definition in float64.

Tolerances.  A bf16 result is rounded once: half a step is 2^-8 of the value.  Before that, in fp32:
cosine and sine are off by less than 2^-22 (the angle's float rounding, sincospi's own last bits), the
products and sum of a pair by 3 * 2^-24, so a rotation is off by at most 2^-21 (|a| + |b|), taken
here as 2^-20 of the head's largest element.  For bf16 the hardware's sine and cosine are used, which are off by up to
2^-21.2 and would allow 1.5 * 2^-20 where every error points one way; the tolerance stays at 2^-20.  The norm's mean of squares adds at most 21 roundings in a
chain (16 elements a lane, five shuffles) and rsqrt two, 2^-19 in all, halved by the square root.  The
input gradient combines three such terms: 2^-17 of the tensor's largest element.  A weight gradient
is a sum of n products, each off by 2^-19, with a chain of at most n additions: (2^-19 + n 2^-24) of
the sum of the products' absolute values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
F32 = torch.float32


def case(B, L, Hq, Hk, D, sections, layout="half", order="blocks", spectrum="axis", dtype=BF16, form="packed", pos="shared"):
    return (B, L, Hq, Hk, D, sections, layout, order, spectrum, dtype, form, pos)


CASES = [
    case(2, 50, 3, 3, 64, (16, 16)),
    case(1, 1, 1, 1, 2, (1,)),
    case(16, 1, 32, 8, 128, (64,), pos="batch"),
    case(3, 17, 4, 2, 128, (16, 24, 24), spectrum="shared", dtype=F32),
    case(2, 33, 5, 1, 80, (20, 12), layout="interleaved", order="cycled"),
    case(2, 9, 2, 2, 70, (35,), dtype=BF16),                                   # odd pairs: element by element
    case(2, 9, 2, 2, 70, (11, 6, 4), layout="interleaved", dtype=F32),
    case(1, 40, 3, 1, 36, (9, 9), order="cycled"),
    case(1, 21, 2, 1, 72, (18, 12), dtype=BF16, form="plain"),                 # two-pair vectors
    case(1, 70, 1, 1, 512, (100, 156), spectrum="shared"),
    case(1, 13, 7, 1, 512, (255,), dtype=F32),
    case(2, 19, 4, 4, 96, (8, 8, 8), form="heads_first"),
    case(2, 65, 6, 2, 256, (64, 64), form="offset", dtype=BF16),               # base not 16-byte aligned
    case(1, 3000, 3, 3, 64, (16, 16), dtype=F32, pos="int32"),
    case(4, 2500, 8, 2, 128, (64,), pos="batch"),                              # several tiles per block
]


def ids(c):
    return f"{c[0]}x{c[1]}-{c[2]}+{c[3]}x{c[4]}-{'.'.join(map(str, c[5]))}-{c[6]}-{str(c[9])[6:]}-{c[10]}-{c[11]}"


def make_heads(gen, B, L, Hq, Hk, D, dtype, form):
    def rand(*s):
        return torch.randn(*s, generator=gen).to(dtype).cuda()
    if form == "packed":
        x = rand(B, L, (Hq + 2 * Hk) * D)
        return x[..., :Hq * D].view(B, L, Hq, D), x[..., Hq * D:(Hq + Hk) * D].view(B, L, Hk, D)
    if form == "heads_first":
        return rand(B, Hq, L, D).transpose(1, 2), rand(B, Hk, L, D).transpose(1, 2)
    if form == "offset":
        return (rand(B * L * Hq * D + 1)[1:].view(B, L, Hq, D), rand(B * L * Hk * D + 1)[1:].view(B, L, Hk, D))
    return rand(B, L, Hq, D), rand(B, L, Hk, D)


def make_positions(gen, B, L, axes, pos):
    p = torch.randint(0, 5000, (L, axes), generator=gen)
    if pos == "batch":
        p = p[None] + torch.randint(-3000, 120000, (B, 1, 1), generator=gen)
    return (p.to(torch.int32) if pos == "int32" else p).cuda()


def spectrum_of(sections, order, spectrum, base):
    """(axis, radians per position) of every pair, restated."""
    if order == "blocks":
        axis = sum(([a] * n for a, n in enumerate(sections)), [])
    else:
        axis, j = [], 0
        while len(axis) < sum(sections):
            axis += [a for a, n in enumerate(sections) if n > j]
            j += 1
    freq = []
    for p, a in enumerate(axis):
        nth = axis[:p].count(a)
        freq.append(base ** -(nth / sections[a]) if spectrum == "axis" else base ** -(p / sum(sections)))
    return axis, freq


def turn64(x, positions, axis, freq, layout):
    n = len(axis)
    ang = positions.double()[..., axis] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = ang.cos().unsqueeze(-2), ang.sin().unsqueeze(-2)
    y = x.clone()
    ia = torch.arange(n) if layout == "half" else 2 * torch.arange(n)
    ib = ia + n if layout == "half" else ia + 1
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    return y


def close(got, want, dtype, atol):
    want = want.to(got.device)
    rtol = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    err = (got.double() - want).abs()
    bad = err > rtol * want.abs() + atol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, largest {float(err.max()):.3e}"


def setup(c, seed=0):
    from custom import RotaryPositions
    B, L, Hq, Hk, D, sections, layout, order, spectrum, dtype, form, pos = c
    gen = torch.Generator().manual_seed(seed + B + 7 * L + D)
    q, k = make_heads(gen, B, L, Hq, Hk, D, dtype, form)
    p = make_positions(gen, B, L, len(sections), pos)
    rot = RotaryPositions(D, sections, base=1000.0, layout=layout, order=order, spectrum=spectrum).cuda()
    axis, freq = spectrum_of(sections, order, spectrum, 1000.0)
    return gen, q, k, p, rot, lambda x, sign=1: turn64(x, p * sign, axis, freq, layout)


@pytest.mark.parametrize("c", CASES, ids=ids)
def test_rotary_forward_and_backward(c):
    gen, q, k, p, rot, turn = setup(c)
    dtype = c[9]
    q.requires_grad_()
    k.requires_grad_()
    outs = rot(q, k, positions=p)
    grads = [torch.randn(o.shape[0], o.shape[2], o.shape[1], o.shape[3], generator=gen).to(dtype).cuda().transpose(1, 2) for o in outs]
    dx = torch.autograd.grad(outs, [q, k], grads)
    for x, o, g, d in zip((q, k), outs, grads, dx):
        assert o.shape == x.shape and o.dtype == dtype and d.shape == x.shape
        close(o, turn(x.detach().double()), dtype, 2.0 ** -20 * float(x.detach().abs().max()))
        close(d, turn(g.double(), -1), dtype, 2.0 ** -20 * float(g.abs().max()))
    one = rot(q, positions=p)
    assert torch.equal(one, outs[0])


@pytest.mark.parametrize("c", CASES, ids=ids)
def test_qk_norm_rotary_forward_and_backward(c):
    from custom import FusedQKNorm
    gen, q, k, p, rot, turn = setup(c, seed=3)
    D, dtype = c[4], c[9]
    mod = FusedQKNorm(D, rotary=rot, eps=1e-6).cuda()
    with torch.no_grad():
        mod.q_weight.copy_(1.0 + 0.3 * torch.randn(D, generator=gen))
        mod.k_weight.copy_(1.0 + 0.3 * torch.randn(D, generator=gen))
    q.requires_grad_()
    k.requires_grad_()
    outs = mod(q, k, p)
    grads = [torch.randn(o.shape, generator=gen).to(dtype).cuda() for o in outs]
    dq, dk, dwq, dwk = torch.autograd.grad(outs, [q, k, mod.q_weight, mod.k_weight], grads)
    for x, o, g, dx, dw, wp in zip((q, k), outs, grads, (dq, dk), (dwq, dwk), (mod.q_weight, mod.k_weight)):
        x64, w = x.detach().double(), wp.detach().double()
        r = 1.0 / (x64.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        xh = x64 * r
        want = turn(w * xh)
        close(o, want, dtype, 2.0 ** -19 * float(want.abs().max()))
        gb = turn(g.double(), -1)
        u = gb * w
        wdx = r * (u - xh * (u * xh).mean(-1, keepdim=True))
        # the terms may cancel: the bound is on them, not on their difference
        scale = float((r * (u.abs() + xh.abs() * (u * xh).abs().mean(-1, keepdim=True))).max())
        close(dx, wdx, dtype, 2.0 ** -17 * scale)
        n = x.shape[0] * x.shape[1] * x.shape[2]
        err = (dw.double() - (gb * xh).sum((0, 1, 2))).abs()
        assert (err <= (2.0 ** -19 + n * 2.0 ** -24) * (gb * xh).abs().sum((0, 1, 2)) + 1e-30).all()
        # reproducible
    again = torch.autograd.grad(mod(q, k, p), [q, k, mod.q_weight, mod.k_weight], grads)
    assert all(torch.equal(a, b) for a, b in zip(again, (dq, dk, dwq, dwk)))


def test_norm_without_positions_and_zero_rows():
    from custom import FusedQKNorm
    mod = FusedQKNorm(64, eps=1e-4).cuda()
    x = torch.randn(2, 5, 3, 64, device="cuda")
    x[0, 1] = 0.0
    q = x.clone().requires_grad_()
    k = x[:, :, :1].clone().requires_grad_()
    yq, yk = mod(q, k)
    want = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-4).sqrt()
    close(yq.detach(), want, F32, 2.0 ** -19 * float(want.abs().max()))
    assert (yq[0, 1] == 0).all()
    g = torch.randn_like(x)
    (dq,) = torch.autograd.grad(yq, q, g)
    close(dq[0, 1], g[0, 1].double() * 100.0, F32, 2.0 ** -17 * 500.0)      # 1 / sqrt(eps) of the gradient
    assert yk.shape == k.shape


@pytest.mark.parametrize("base", [0, 1_000_000, 2 ** 31 + 5, -7_000_000, 2 ** 45 + 1])
def test_far_and_negative_positions(base):
    """The angle wraps exactly.  The want is built from exact integer arithmetic: a position's multiple
    of a frequency given as a multiple of 2^-20 turns."""
    from custom import RotaryPositions
    num = [1, 3, 77777, 524287, 2 ** 19, 2 ** 18, 13, 1048575]
    rot = RotaryPositions(16, (8,), frequencies=[2.0 * math.pi * n / 2 ** 20 for n in num], layout="interleaved").cuda()
    pos = torch.arange(base, base + 300)
    x = torch.zeros(1, 300, 1, 16)
    x[..., 0::2] = 1.0
    got = rot(x.cuda(), positions=pos.cuda()).double().cpu()
    frac = torch.tensor([[(int(q) * n) % 2 ** 20 for n in num] for q in pos], dtype=torch.float64) / 2 ** 20 * (2.0 * math.pi)
    # f / 2 pi is rounded to 53 bits, 2^-54 of a turn at most, times the position; the rest is fp32
    tol = 2.0 ** -21 + 2.0 * math.pi * abs(base + 300) * 2.0 ** -53
    tol = min(tol, 2.0)
    assert (got[0, :, 0, 0::2] - frac.cos()).abs().max() <= tol
    assert (got[0, :, 0, 1::2] - frac.sin()).abs().max() <= tol


def test_gradients_against_differences():
    from custom import FusedQKNorm, RotaryPositions
    rot = RotaryPositions(32, (8, 8), base=100.0).cuda()
    mod = FusedQKNorm(32, rotary=rot, eps=1e-3).cuda()
    gen = torch.Generator().manual_seed(1)
    q, k = torch.randn(2, 6, 3, 32, generator=gen).cuda(), torch.randn(2, 6, 1, 32, generator=gen).cuda()
    p = torch.randint(0, 40, (6, 2), generator=gen).cuda()
    gq, gk = torch.randn(q.shape, generator=gen).cuda(), torch.randn(k.shape, generator=gen).cuda()
    leaves = [q, k, mod.q_weight.detach().clone(), mod.k_weight.detach().clone()]

    def f(q, k, wq, wk):
        with torch.no_grad():
            mod.q_weight.copy_(wq)
            mod.k_weight.copy_(wk)
            a, b = mod(q, k, p)
        return float((a.double() * gq).sum() + (b.double() * gk).sum())

    q.requires_grad_()
    k.requires_grad_()
    grads = torch.autograd.grad(mod(q, k, p), [q, k, mod.q_weight, mod.k_weight], [gq, gk])
    h = 2.0 ** -7
    for i in range(4):
        d = torch.randn(leaves[i].shape, generator=gen).cuda()
        plus, minus = [t.detach().clone() for t in leaves], [t.detach().clone() for t in leaves]
        plus[i] += h * d
        minus[i] -= h * d
        got = (f(*plus) - f(*minus)) / (2 * h)
        want = float((grads[i].double() * d).sum())
        # rounding of the two sums of ~768 outputs of size ~1: 2^-21 * 28 / h; the third derivative times h^2 / 6
        assert abs(got - want) <= 28 * 2.0 ** -21 / h + 50 * h * h + 1e-3 * abs(want), i
        f(*leaves)


def test_empty_and_broadcast():
    from custom import FusedQKNorm, RotaryPositions
    rot = RotaryPositions(64, (32,)).cuda()
    mod = FusedQKNorm(64, rotary=rot).cuda()
    for B, L in ((0, 4), (3, 0)):
        q = torch.zeros(B, L, 2, 64, device="cuda", requires_grad=True)
        k = torch.zeros(B, L, 1, 64, device="cuda", requires_grad=True)
        p = torch.zeros(L, 1, dtype=torch.int64, device="cuda")
        a, b = mod(q, k, p)
        assert a.shape == q.shape and b.shape == k.shape
        g = torch.autograd.grad((a.sum() + b.sum()), [q, k, mod.q_weight, mod.k_weight])
        assert (g[2] == 0).all() and (g[3] == 0).all()
    # an expanded input, an expanded gradient (sum), one position for all tokens of a batch
    base = torch.randn(1, 7, 1, 64, device="cuda", requires_grad=True)
    x = base.expand(3, 7, 4, 64)
    pos = torch.arange(7, device="cuda").unsqueeze(-1)
    y = rot(x, positions=pos)
    assert torch.equal(y[0, :, 0], y[2, :, 3])
    (g,) = torch.autograd.grad(y.sum(), base)
    ones = rot(torch.ones(1, 7, 1, 64, device="cuda"), positions=-pos)
    assert torch.allclose(g, 12 * ones, rtol=1e-5, atol=1e-4)
    t = torch.randn(7, 4, 64, device="cuda")
    assert torch.equal(rot(t, positions=pos), rot(t[None], positions=pos)[0])


def test_in_place_through_the_c_entry():
    import ctypes

    from backend import _lib
    from custom import RotaryPositions
    rot = RotaryPositions(64, (16, 16)).cuda()
    x = torch.randn(2, 30, 3, 64, device="cuda")
    p = torch.randint(0, 99, (30, 2), device="cuda")
    want = rot(x, positions=p)
    arr = (ctypes.c_int64 * 5)(x.data_ptr(), 3, 30 * 3 * 64, 3 * 64, 64)
    turns, axis, axes, interleaved = rot.table
    r = _lib.Rotary(p.data_ptr(), 1, 0, p.stride(0), p.stride(1), axes, turns.numel(), int(interleaved), turns.data_ptr(), axis.data_ptr())
    _lib.check(_lib.lib().fp4t_rotary(arr, arr, 1, _lib.DT_F32, 2, 30, 64, ctypes.byref(r), 0, _lib.stream_ptr(x.device)), "fp4t_rotary")
    assert torch.equal(x, want)


def test_side_stream_and_graph_replay():
    from custom import FusedQKNorm, RotaryPositions
    rot = RotaryPositions(64, (16, 16), base=100.0).cuda()
    mod = FusedQKNorm(64, rotary=rot).cuda()
    p = torch.randint(0, 50, (50, 2), device="cuda")

    def step(q, k, gq, gk):
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = mod(q, k, p)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, [q, k, mod.q_weight, mod.k_weight], [gq, gk]))

    def data(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return [torch.randn(64, 50, 3, 64, device="cuda", generator=g, dtype=F32).to(BF16) for _ in range(4)]

    static = data(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step(*static)))
    graphs = []
    for _ in range(2):                       # two graphs, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, out))
    for seed in (1, 2):
        fresh = data(seed)
        want = step(*fresh)
        for s, f in zip(static, fresh):
            s.copy_(f)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (g, _), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals_on_the_gpu():
    from custom import FusedQKNorm, RotaryPositions
    rot = RotaryPositions(64, (16, 16)).cuda()
    x = torch.zeros(2, 5, 3, 64, device="cuda")
    p = torch.zeros(5, 2, dtype=torch.int64, device="cuda")
    for bad in (p[:4], p[:, :1], p.float(), p[:, 0], p[None].expand(3, 5, 2), p.cpu()):
        with pytest.raises((ValueError, NotImplementedError)):
            rot(x, positions=bad)
    for y in (x.half(), x.double(), x[..., :32], x[0, 0], x.cpu()):
        with pytest.raises((ValueError, NotImplementedError)):
            rot(y, positions=p)
    with pytest.raises(ValueError):
        rot(x, x.bfloat16(), positions=p)
    with pytest.raises(ValueError):
        rot(x, x[:, :4], positions=p)
    mod = FusedQKNorm(64, rotary=rot).cuda()
    with pytest.raises(ValueError):
        mod(x, x)
    with pytest.raises(ValueError):
        FusedQKNorm(64).cuda()(x, x, p)


def test_parametrized_weights():
    """A parametrized weight is used as parametrized, and its gradient goes through the parametrization."""
    from custom import FusedQKNorm

    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    gen = torch.Generator().manual_seed(3)
    q = torch.randn(2, 9, 3, 64, generator=gen).cuda()
    plain, made = FusedQKNorm(64).cuda(), FusedQKNorm(64).cuda()
    torch.nn.utils.parametrize.register_parametrization(made, "q_weight", Twice())
    with torch.no_grad():
        plain.q_weight.fill_(2.0)
    want, got = plain(q, q), made(q, q)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    original = made.parametrizations.q_weight.original
    dwant, = torch.autograd.grad(want[0].square().sum(), plain.q_weight)
    dgot, = torch.autograd.grad(got[0].square().sum(), original)
    assert torch.equal(2 * dwant, dgot)                  # a factor of two is exact
