"""Linear cross entropy (fp4t_linear_xent_forward / _backward) against the definition in float64 on the same
bf16 operands.

Tolerances are bounds, elementwise.  A logit is a sum of D products accumulated in fp32: off by at most
ex = D 2^-23 max(|h| |w|^T).  The losses add the exponentials' and the sum's roundings, 2^-18 of the
terms and of the value.  dl is off by p g (2 ex + 2^-17) and by its rounding to bf16, half a step, 2^-8 |dl| (2^-16 up to 64
tokens, where it is kept in two bf16); the products carry that into dh and dW through |W| and |h|, add their own accumulation, n 2^-23 of the
terms' absolute sum, and (bf16 results) half a step of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32

# tokens, dim, vocab, bias dtype, reduction, share of ignored tokens
CASES = [
    (1, 8, 1, None, "mean", 0.0),
    (1, 64, 10, F32, "sum", 0.0),
    (3, 72, 7, BF16, "none", 0.0),
    (512, 192, 10, F32, "mean", 0.0),
    (130, 64, 1000, None, "mean", 0.3),
    (257, 136, 300, BF16, "sum", 0.0),
    (300, 128, 513, F32, "none", 0.5),
    (128, 256, 128, None, "mean", 0.0),
    (256, 512, 256, None, "mean", 0.1),
    (255, 520, 4097, BF16, "mean", 0.0),
    (2, 4096, 2000, None, "none", 0.0),
    (5000, 64, 33, F32, "mean", 0.2),          # dW split over the tokens
    (40, 64, 50001, F32, "mean", 0.0),         # dh split over the vocabulary
    (1111, 1032, 777, None, "sum", 0.9),
    (40000, 64, 9000, BF16, "mean", 0.1),      # several blocks of tokens, several pieces of the vocabulary
    (20000, 8, 27000, None, "mean", 0.0),      # pieces and splits together
    (20000, 16, 27000, F32, "none", 0.7),      # the same with most tokens ignored: whole blocks of slots are empty
    (33000, 64, 500, None, "mean", 0.995),     # a few slots left of many tokens; per-run counts
    (3, 64, 500, None, "sum", 0.7),
    (63, 192, 1000, BF16, "mean", 0.0),
    (64, 64, 5000, F32, "none", 0.0),
    (64, 200, 130, F32, "sum", 0.5),
    (65, 200, 130, F32, "sum", 0.5),
    (7, 20000, 100, None, "mean", 0.0),        # more column tiles than clusters to split over
]


def make(T, D, V, bias, ignored, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + T + D + V)
    h = (torch.randn(T, D, generator=g) * scale).to(BF16).cuda()
    w = (torch.randn(V, D, generator=g) / D ** 0.5).to(BF16).cuda()
    b = None if bias is None else (torch.randn(V, generator=g) * 0.3).to(bias).cuda()
    t = torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) < ignored] = -100
    return h, w, b, t.cuda()


def reference(h, w, b, t, reduction, grad):
    """float64 loss and gradients, and the bounds of the module's docstring."""
    H, W = h.double(), w.double()
    D, V, T = H.shape[1], W.shape[0], H.shape[0]
    x = H @ W.T + (0 if b is None else b.double())
    keep = t != -100
    y = t.clamp_min(0)[:, None]
    lse = torch.logsumexp(x, 1)
    loss = torch.where(keep, lse - x.gather(1, y)[:, 0], 0.0)
    n = keep.sum()
    out = loss if reduction == "none" else loss.sum() / (n if reduction == "mean" else 1)
    gr = grad.double() / (n if reduction == "mean" else 1)
    gr = torch.where(keep, gr, 0.0)[:, None].expand(T, 1)
    p = x.sub_(lse[:, None]).exp_()
    ex = D * 2.0 ** -23 * float((H.abs() @ W.abs().T).max())
    e = p * gr.abs() * (2 * ex + 2.0 ** -17)
    eb = e.sum(0)                                # db is summed before the rounding
    dl = p.mul_(gr).scatter_add_(1, y, -gr)
    e += dl.abs() * (2.0 ** -16 if T <= 64 else 2.0 ** -8)
    res = {"loss": out, "loss_tol": (2 * ex + 2.0 ** -18) * (1 if reduction != "sum" else max(1, int(n))) + 2.0 ** -18 * out.abs()}
    res["dh"], res["dw"], res["db"] = dl @ W, dl.T @ H, dl.sum(0)
    a = dl.abs_()
    res["dh_tol"] = e @ W.abs() + V * 2.0 ** -23 * (a @ W.abs())
    res["dw_tol"] = e.T @ H.abs() + T * 2.0 ** -23 * (a.T @ H.abs())
    res["db_tol"] = eb + T * 2.0 ** -23 * a.sum(0)
    return res


def within(got, want, tol, what):
    if got.dtype == BF16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    else:
        tol = tol + 2.0 ** -23 * want.abs()
    bad = ~((got.double() - want).abs() <= tol + 1e-37)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max()):.3e}"


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{str(c[3])[6:]}-{c[4]}-{c[5]}")
def test_loss_and_gradients(case):
    from backend import ops
    from custom import linear_cross_entropy
    T, D, V, bias, reduction, ignored = case
    h, w, b, t = make(T, D, V, bias, ignored)
    grad = (torch.rand(T, device="cuda") + 0.5) if reduction == "none" else torch.tensor(0.75, device="cuda")
    want = reference(h, w, b, t, reduction, grad)
    leaves = [x.requires_grad_() for x in (h, w, b) if x is not None]
    loss = linear_cross_entropy(h, w, t, b, reduction=reduction)
    assert loss.dtype == F32 and loss.shape == want["loss"].shape
    grads = torch.autograd.grad(loss, leaves, grad)
    within(loss.detach(), want["loss"], want["loss_tol"], "loss")
    for got, leaf, name in zip(grads, leaves, ("dh", "dw", "db")):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        within(got, want[name], want[name + "_tol"], name)
    if ignored:
        assert (grads[0][t == -100] == 0).all()
    # reproducible, and each gradient alone is the same
    assert all(torch.equal(x, y) for x, y in zip(grads, torch.autograd.grad(linear_cross_entropy(h, w, t, b, reduction=reduction), leaves, grad)))
    hd, wd = h.detach(), w.detach()
    bd = None if b is None else b.detach()
    _, lse, count = ops.linear_cross_entropy_forward(hd, wd, bd, t, -100, reduction)
    assert float(count) == int((t != -100).sum())
    only = ops.linear_cross_entropy_backward(grad, hd, wd, bd, t, lse, -100, reduction, dw_dtype=BF16)
    assert only[0] is None and only[2] is None and torch.equal(only[1], grads[1])
    ops.check_status()


def test_fp32_gradients_under_autocast():
    from custom import linear_cross_entropy
    h, w, b, t = make(300, 192, 1000, F32, 0.1)
    want = reference(h, w, b, t, "mean", torch.tensor(1.0, device="cuda"))
    hf, wf = h.float().requires_grad_(), w.float().requires_grad_()
    b.requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        loss = linear_cross_entropy(hf.view(30, 10, 192), wf, t.view(30, 10), b)
    grads = torch.autograd.grad(loss, [hf, wf, b])
    for got, name in zip(grads, ("dh", "dw", "db")):
        assert got.dtype == F32
        within(got, want[name], want[name + "_tol"], name)


def test_gradients_against_differences():
    """Directional differences of the float64 mean of the kernel's own fp32 losses, along bf16 steps that
    leave the operands exact: h, w in multiples of 2^-4, steps of 2^-4."""
    from custom import linear_cross_entropy
    g = torch.Generator().manual_seed(3)
    T, D, V = 90, 64, 200

    def grid(*s):
        return torch.randint(-12, 13, s, generator=g).float() / 16
    h, w = grid(T, D), grid(V, D)
    dh, dw = torch.randint(-1, 2, (T, D), generator=g).float() / 16, torch.randint(-1, 2, (V, D), generator=g).float() / 16
    t = torch.randint(0, V, (T,), generator=g).cuda()
    grad = (torch.rand(T, generator=g) + 0.5).cuda()

    def f(a, b):
        return float((linear_cross_entropy((h + a * dh).to(BF16).cuda(), (w + b * dw).to(BF16).cuda(), t, reduction="none").double() * grad).sum())
    hl, wl = h.to(BF16).cuda().requires_grad_(), w.to(BF16).cuda().requires_grad_()
    gh, gw = torch.autograd.grad(linear_cross_entropy(hl, wl, t, reduction="none"), [hl, wl], grad)
    for a, b, want in ((1, 0, (gh.double().cpu() * dh).sum()), (0, 1, (gw.double().cpu() * dw).sum())):
        # fourth-order central difference over whole steps: the error is the fifth derivative over 30.
        # Along this direction a logit moves by z, |z| <= sum |h| |dw| ~ 64 * 0.37 * 0.04: rms 0.25, so the
        # fifth cumulants are below 0.25^5 * 10 a token, 0.01 * 90 / 30 in all; the gradients' bf16 roundings
        # are independent: 2^-8 of the root of the sum of squares, 4 deviations, and 2^-8 of it coherently.
        got = (8 * (f(a, b) - f(-a, -b)) - (f(2 * a, 2 * b) - f(-2 * a, -2 * b))) / 12
        root = float(((gh.double().cpu() * dh) if a else (gw.double().cpu() * dw)).norm())
        assert abs(got - float(want)) <= 0.03 + 5 * 2.0 ** -8 * root + 2.0 ** -8 * abs(float(want))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_all_tokens_ignored_and_no_tokens(reduction):
    from custom import linear_cross_entropy
    h, w, b, t = make(70, 64, 300, F32, 0.0)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    loss = linear_cross_entropy(h, w, torch.full_like(t, -100), b, reduction=reduction)
    assert loss.isnan().all() if reduction == "mean" else (loss == 0).all()
    for g in torch.autograd.grad(loss, leaves, torch.ones_like(loss)):
        assert (g == 0).all()
    loss = linear_cross_entropy(h[:0], w, t[:0], b, reduction=reduction)
    assert loss.shape == ((0,) if reduction == "none" else ())
    assert reduction == "none" or (loss.isnan() if reduction == "mean" else loss == 0)
    for g in torch.autograd.grad(loss, leaves, torch.ones_like(loss)):
        assert (g == 0).all()


def test_masked_entries_infinities_and_nan():
    """A bias of -inf takes entries out (all of a tile too); NaN and infinities stay in their rows' losses; a
    masked token's garbage does not reach the others."""
    from custom import linear_cross_entropy
    T, D, V = 200, 64, 700
    h, w, _, t = make(T, D, V, None, 0.0)
    b = torch.zeros(V, device="cuda")
    b[:300] = -float("inf")
    t = 300 + t % 400
    want = torch.nn.functional.cross_entropy(h.double() @ w[300:].double().T, t - 300, reduction="none")
    got = linear_cross_entropy(h, w, t, b, reduction="none")
    assert (got.double() - want).abs().max() <= 2 * 64 * 2.0 ** -23 * 40 + 2.0 ** -18 * 10
    hl, wl, bl = h.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    gh, gw, gb = torch.autograd.grad(linear_cross_entropy(hl, wl, t, bl), [hl, wl, bl])
    assert (gw[:300] == 0).all() and (gb[:300] == 0).all() and gh.isfinite().all()
    low = b.clone()
    low[:300] = torch.finfo(F32).min
    assert bool((linear_cross_entropy(h, w, t, low, reduction="none") == got).all())
    # a row that the lowest value masks altogether: uniform, as its softmax is
    uniform = linear_cross_entropy(hl, wl, t, torch.full_like(b, torch.finfo(F32).min), reduction="none")
    assert (uniform - torch.log(torch.tensor(700.0, device="cuda"))).abs().max() <= 2.0 ** -20 * torch.finfo(F32).max
    (gu,) = torch.autograd.grad(uniform.sum(), hl)
    assert gu.isfinite().all()
    target_masked = t.clone()
    target_masked[5] = 7
    assert linear_cross_entropy(h, w, target_masked, b, reduction="none")[5] == float("inf")
    assert linear_cross_entropy(h, w, t, torch.full_like(b, -float("inf")), reduction="none").isnan().all()
    bad = h.clone()
    bad[3] = float("nan")
    bad[4] = float("inf")
    t2 = t.clone()
    t2[3:5] = -100
    out = linear_cross_entropy(bad, w, t2, b, reduction="none")
    assert (out[3:5] == 0).all() and torch.equal(out[5:], got[5:])
    # the ignored tokens' garbage reaches no gradient: as if they were not there
    for dt in (BF16, F32):
        bl2 = b.clone().requires_grad_()
        with torch.autocast("cuda", dtype=BF16):
            got1 = torch.autograd.grad(linear_cross_entropy(bad.to(dt).requires_grad_(), wl, t2, bl2), [wl, bl2])
            leaf = bad.to(dt).requires_grad_()
            (got2,) = torch.autograd.grad(linear_cross_entropy(leaf, wl, t2, b), leaf)
            keep = torch.cat([torch.arange(3), torch.arange(5, T)]).cuda()
            rest = h[keep].to(dt).requires_grad_()
            want1 = torch.autograd.grad(linear_cross_entropy(rest, wl, t[keep], bl2), [rest, wl, bl2])
        assert torch.equal(got1[0], want1[1]) and torch.equal(got1[1], want1[2])
        assert (got2[3:5] == 0).all() and torch.equal(got2[keep], want1[0])
    out = linear_cross_entropy(bad, w, t, b, reduction="none")
    assert out[3].isnan() and out[4].isnan() and torch.equal(out[5:], got[5:])


def test_large_logits():
    """Logits of a few hundred: the running maximum carries over tiles in both directions."""
    from custom import linear_cross_entropy
    h, w, b, t = make(140, 128, 2000, F32, 0.0, scale=100.0)
    order = (h[0].double() @ w.double().T).argsort()
    for perm in (order, order.flip(0)):
        wp = w[perm].contiguous()
        want = reference(h, wp, b, t, "none", torch.ones(140, device="cuda"))
        within(linear_cross_entropy(h, wp, t, b, reduction="none"), want["loss"], want["loss_tol"], "loss")


def test_target_outside_the_vocabulary_is_reported():
    from backend import ops
    from custom import linear_cross_entropy
    h, w, b, t = make(20, 64, 50, None, 0.0)
    good = linear_cross_entropy(h, w, t, reduction="none")
    for wrong in (50, -1, 2 ** 40, -2 ** 63):
        bad = t.clone()
        bad[4] = wrong
        loss = linear_cross_entropy(h, w, bad, reduction="none")
        assert loss[4].isnan() and torch.equal(loss[5:], good[5:])
        with pytest.raises(RuntimeError, match="outside the vocabulary"):
            ops.check_status()
        ops.check_status()


def test_strides_and_views():
    from custom import linear_cross_entropy
    h, w, b, t = make(64, 64, 200, None, 0.0)
    want = linear_cross_entropy(h, w, t)
    wide = torch.zeros(64, 3, 64, dtype=BF16, device="cuda")
    wide[:, 1] = h
    assert torch.equal(linear_cross_entropy(wide[:, 1], w, t), want)                     # rows 192 apart
    assert torch.equal(linear_cross_entropy(h.T.contiguous().T, w.T.contiguous().T, t), want)
    odd = torch.zeros(64 * 64 + 3, dtype=BF16, device="cuda")[3:].view(64, 64)
    odd.copy_(h)
    assert torch.equal(linear_cross_entropy(odd, w, t), want)
    assert torch.equal(linear_cross_entropy(h.view(4, 16, 64), w, t.view(4, 16)), want)
    same = h[:1].expand(64, 64)
    assert torch.equal(linear_cross_entropy(same, w, t, reduction="none"), linear_cross_entropy(same.contiguous(), w, t, reduction="none"))
    tt = torch.stack([t, t], 1)[:, 0]
    assert torch.equal(linear_cross_entropy(h, w, tt), want)
    assert linear_cross_entropy(h[0], w, t[0]).shape == ()


def test_side_stream_and_graph_replay():
    from custom import linear_cross_entropy

    def step(h, w, b, t):
        leaves = [x.detach().requires_grad_() for x in (h, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))

    static = list(make(300, 192, 1000, F32, 0.2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step(*static)))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, out))
    for seed in (1, 2):
        fresh = make(300, 192, 1000, F32, 0.2, seed=seed)
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
    from custom import linear_cross_entropy
    h, w, b, t = make(16, 64, 50, F32, 0.0)
    for args in ((h.float(), w, t), (h, w.float(), t), (h.half(), w, t), (h, w[:, :56], t), (h[:, :60], w[:, :60], t), (h, w, t[:5]),
                 (h, w, t.int()), (h, w[:0], t), (h, w, t, b[:5]), (h, w, t, b.half()), (h, w, t.cpu()), (h.cpu(), w, t)):
        with pytest.raises((ValueError, NotImplementedError)):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        linear_cross_entropy(h, w, t, reduction="median")
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError):
        linear_cross_entropy(h.float(), w, t)
