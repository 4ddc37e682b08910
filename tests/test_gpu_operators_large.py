"""Rotary, norm and linear cross entropy where element offsets pass 32 bits, and on two streams at once.
Results are compared with the same operator on a part that is small, or with float64 on that part."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _room(gigabytes):
    free, _ = torch.cuda.mem_get_info()
    if free < gigabytes * 2 ** 30:
        pytest.skip(f"needs {gigabytes} GB of device memory")


@pytest.mark.parametrize("form", ["tokens_first", "heads_first"])
def test_rotary_and_norm_past_32_bits(form):
    """330000 tokens x 52 heads x 128: 2.2e9 elements.  The last tokens of the last heads equal those of a call on
    them alone (every head's result depends on its own elements and position only)."""
    from custom import FusedQKNorm, RotaryPositions
    _room(40)
    L, H, D = 330_000, 52, 128
    gen = torch.Generator(device="cuda").manual_seed(0)
    part = torch.randn(1, 300, H, D, device="cuda", generator=gen).to(BF16)
    gpart = torch.randn(1, 300, H, D, device="cuda", generator=gen).to(BF16)
    shape = (1, L, H, D) if form == "tokens_first" else (1, H, L, D)
    x, g = torch.zeros(shape, dtype=BF16, device="cuda"), torch.zeros(shape, dtype=BF16, device="cuda")
    if form == "heads_first":
        x, g = x.transpose(1, 2), g.transpose(1, 2)
    assert x.numel() > 2 ** 31
    x[:, -300:] = part
    g[:, -300:] = gpart
    pos = torch.arange(L, device="cuda").unsqueeze(-1)
    rot = RotaryPositions(D, (64,)).cuda()
    norm = FusedQKNorm(D, rotary=rot, eps=1e-3).cuda()
    y = rot(x, positions=pos)
    assert torch.equal(y[:, -300:], rot(part, positions=pos[-300:])) and (y[:, :300] == 0).all()
    del y
    x.requires_grad_()
    part.requires_grad_()
    k, pk = x[:, :, -1:].detach(), part[:, :, -1:].detach()
    yq, yk = norm(x, k, pos)
    zq, zk = norm(part, pk, pos[-300:])
    assert torch.equal(yq[:, -300:], zq) and torch.equal(yk[:, -300:], zk)
    dx, dw = torch.autograd.grad(yq, [x, norm.q_weight], g)
    px, pw = torch.autograd.grad(zq, [part, norm.q_weight], gpart)
    assert torch.equal(dx[:, -300:], px) and (dx[:, :300] == 0).all()
    # the same 15600 terms in another association: bounded by 2^-24 times a chain of as many
    assert ((dw - pw).abs() <= 15600 * 2.0 ** -24 * 4 * 15600 ** 0.5 + 1e-3).all()


def test_linear_cross_entropy_past_32_bits():
    """280000 entries x 8192: W and dW have 2.3e9 elements.  float64 in pieces of the vocabulary."""
    from custom import linear_cross_entropy
    _room(40)
    T, D, V = 40, 8192, 280_000
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(T, D, device="cuda", generator=gen).to(BF16).requires_grad_()
    w = torch.empty(V, D, dtype=BF16, device="cuda")
    assert w.numel() > 2 ** 31
    for i in range(0, V, 40_000):
        w[i:i + 40_000] = torch.randn(40_000, D, device="cuda", generator=gen) / D ** 0.5
    w.requires_grad_()
    t = torch.randint(0, V, (T,), device="cuda", generator=gen)
    t[-1] = V - 1
    loss = linear_cross_entropy(h, w, t)
    dh, dw = torch.autograd.grad(loss, [h, w])
    hd, wd = h.detach(), w.detach()
    x = torch.cat([hd.double() @ wd[i:i + 20_000].double().T for i in range(0, V, 20_000)], 1)
    lse = torch.logsumexp(x, 1)
    want = (lse - x.gather(1, t[:, None])[:, 0]).mean()
    ex = D * 2.0 ** -23 * float((hd.double().abs() @ wd[:2000].double().abs().T).max())      # bound of a logit's accumulation
    assert abs(float(loss.detach()) - float(want)) <= 2 * ex + 2.0 ** -18 * float(want)
    dl = (x - lse[:, None]).exp_().scatter_add_(1, t[:, None], torch.full((T, 1), -1.0, dtype=torch.float64, device="cuda")) / T
    wdh = sum(dl[:, i:i + 20_000] @ wd[i:i + 20_000].double() for i in range(0, V, 20_000))
    # dl is kept in two bf16 here: the results' own rounding, and the logits' error in the probabilities
    assert (dh.double() - wdh).abs().max() <= (2.0 ** -8 + 2 * ex + 2.0 ** -14) * float(wdh.abs().max())
    for rows in (slice(0, 500), slice(V - 500, V)):
        wdw = dl[:, rows].T @ hd.double()
        bound = (2.0 ** -8 + 2 * ex + 2.0 ** -14) * (dl[:, rows].abs().T @ hd.double().abs())
        assert ((dw[rows].double() - wdw).abs() <= bound + 1e-12).all()


def test_two_streams_at_once():
    """The same calls on two streams with other inputs, not waiting for each other: as one after the other."""
    from custom import FusedQKNorm, RotaryPositions, linear_cross_entropy
    rot = RotaryPositions(64, (16, 16), base=100.0).cuda()
    norm = FusedQKNorm(64, rotary=rot).cuda()
    pos = torch.randint(0, 50, (50, 2), device="cuda")

    def data(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)  # noqa: E731
        return r(64, 50, 3, 64), r(64, 50, 3, 64), r(700, 192), r(5000, 192) * 0.1, torch.randint(0, 5000, (700,), device="cuda", generator=g)

    def step(q, k, h, w, t):
        q, k, h, w = (x.detach().requires_grad_() for x in (q, k, h, w))
        a, b = norm(q, k, pos)
        loss = linear_cross_entropy(h, w, t)
        return [loss.detach()] + list(torch.autograd.grad(loss + a.float().square().sum() + b.float().sum(), [q, k, h, w, norm.q_weight]))

    inputs = [data(0), data(1)]
    want = [step(*d) for d in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_many_sizes_in_a_row():
    """Forty odd shapes one after the other in one process, workspaces coming and going: each as by itself."""
    from custom import linear_cross_entropy
    rng = torch.Generator().manual_seed(5)
    for i in range(40):
        T, D, V = (int(torch.randint(1, n, (1,), generator=rng)) for n in (700, 40, 3000))
        D *= 8
        h = torch.randn(T, D, generator=rng).to(BF16).cuda()
        w = (torch.randn(V, D, generator=rng) / D ** 0.5).to(BF16).cuda()
        t = torch.randint(0, V, (T,), generator=rng).cuda()
        t[torch.rand(T, generator=rng).cuda() < 0.3] = -100
        got = linear_cross_entropy(h, w, t, reduction="none")
        x = h.double() @ w.double().T
        want = torch.nn.functional.cross_entropy(x, t, reduction="none")
        ex = D * 2.0 ** -23 * float((h.double().abs() @ w.double().abs().T).max())
        assert ((got.double() - want).abs() <= 2 * ex + 2.0 ** -18 * (1 + want.abs())).all(), (T, D, V)
