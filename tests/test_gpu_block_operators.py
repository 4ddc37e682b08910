"""Rotary positions, query / key norms and the head's loss together, as the image model uses them: values and
gradients against the same model written out in float64, a training step with every option, and a step
captured into CUDA graphs."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _fp32_convolution():
    """torch runs the patch embedding's convolution in TF32 (2^-11) unless told otherwise."""
    was = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    yield
    torch.backends.cudnn.allow_tf32 = was


CFG = dict(img_size=28, patch_size=4, embed_dim=192, num_heads=3, mlp_ratio=4.0)


def model64(params, x, rope, qk_norm):
    """Logits of a depth-1 TinyViT (dropout off) from its float64 parameters."""
    p = params
    B, H, dh = x.shape[0], 3, 64
    x = F.conv2d(x, p["patch_embed.weight"], p["patch_embed.bias"], stride=4).flatten(2).transpose(1, 2)
    x = torch.cat([p["cls_token"].expand(B, -1, -1), x], 1) + p["pos_embed"]
    L = x.shape[1]
    y = F.layer_norm(x, (192,), p["encoder.attn.preln.weight"], p["encoder.attn.preln.bias"])
    q, k, v = (F.linear(y, p[f"encoder.attn.{n}_proj.weight"], p[f"encoder.attn.{n}_proj.bias"]).view(B, L, H, dh) for n in "qkv")
    if qk_norm:
        q, k = ((t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * p[f"encoder.attn.qk_norm.{n}_weight"] for n, t in (("q", q), ("k", k)))
    if rope:
        i = torch.arange(49, device=x.device)
        pos = torch.cat([torch.zeros(1, 2, device=x.device), torch.stack([i // 7 + 1, i % 7 + 1], 1)]).double()
        f = 100.0 ** (-torch.arange(16, device=x.device).double() / 16)
        ang = torch.cat([pos[:, :1] * f, pos[:, 1:] * f], 1)[:, None]
        turn = lambda t: torch.cat([t[..., :32] * ang.cos() - t[..., 32:] * ang.sin(), t[..., :32] * ang.sin() + t[..., 32:] * ang.cos()], -1)  # noqa: E731
        q, k = turn(q), turn(k)
    a = torch.softmax(torch.einsum("blhd,bmhd->bhlm", q, k) * math.sqrt(dh), -1)
    y = torch.einsum("bhlm,bmhd->blhd", a, v).reshape(B, L, 192)
    x = x + F.linear(y, p["encoder.attn.o_proj.weight"], p["encoder.attn.o_proj.bias"])
    y = F.layer_norm(x, (192,), p["encoder.ffn.preln.weight"], p["encoder.ffn.preln.bias"])
    y = F.linear(F.gelu(F.linear(y, p["encoder.ffn.up_proj.weight"], p["encoder.ffn.up_proj.bias"])), p["encoder.ffn.down_proj.weight"],
                 p["encoder.ffn.down_proj.bias"])
    return F.linear((x + y)[:, 0], p["mlp_head.weight"], p["mlp_head.bias"])


def rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("sdpa", [False, True])
@pytest.mark.parametrize("rope,qk_norm", [(True, False), (False, True), (True, True)])
def test_model_against_float64(rope, qk_norm, sdpa):
    """fp32, dropout off.  About a dozen layers in a chain, each off by 2^-20 or less (products over at most 768
    terms in fp32, the norms' 2^-19 / 2); the softmax carries an error of the scores, |score| <= 8 here, into
    its weights: 12 * 8 * 2^-20 = 2^-13."""
    from models import TinyViT
    torch.manual_seed(0)
    m = TinyViT(**CFG, linear_impl="torch", rope=rope, qk_norm=qk_norm, sdpa=sdpa).cuda().eval()
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "qk_norm" in n:
                p.mul_(1.0 + 0.2 * torch.randn_like(p))
            elif "_proj.weight" in n:
                p.mul_(0.5)              # keeps the reference's sqrt(dh)-multiplied scores small without the norm
    x = torch.rand(16, 1, 28, 28, device="cuda")
    t = torch.randint(0, 10, (16,), device="cuda")
    params = {n: p.detach().double().requires_grad_() for n, p in m.named_parameters()}
    want = model64(params, x.double(), rope, qk_norm)
    got = m(x)
    assert rel(got.detach(), want.detach()) <= 2.0 ** -13
    g64 = torch.autograd.grad(F.cross_entropy(want, t), list(params.values()))
    g32 = torch.autograd.grad(F.cross_entropy(got, t), list(m.parameters()))
    for (n, _), a, b in zip(m.named_parameters(), g32, g64):
        scale = max(float(b.norm()), 1e-6)          # k's bias is close to irrelevant to a softmax: its gradient is a difference of larger terms
        assert float((a.double() - b).norm()) <= 2.0 ** -12 * scale + 2.0 ** -20, n


def test_loss_with_the_head_inside():
    """model.loss against the loss and gradients of its own bf16 features, in float64 (bounds of one
    rounding of dl and of the results, 2^-8 each, doubled by the sums' spread)."""
    from models import TinyViT
    torch.manual_seed(1)
    m = TinyViT(**CFG, linear_impl="torch", rope=True, qk_norm=True).cuda().eval()
    x = torch.rand(64, 1, 28, 28, device="cuda")
    t = torch.randint(0, 10, (64,), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = m.loss(x, t)
        feats = m.features(x)
    head = (m.mlp_head.weight, m.mlp_head.bias)
    gw, gb = torch.autograd.grad(loss, head)
    f64 = feats.detach().to(torch.bfloat16).double()
    w64 = m.mlp_head.weight.detach().to(torch.bfloat16).double().requires_grad_()
    b64 = m.mlp_head.bias.detach().double().requires_grad_()
    want = F.cross_entropy(F.linear(f64, w64, b64), t)
    hw, hb = torch.autograd.grad(want, (w64, b64))
    assert gw.dtype == torch.float32 and gb.dtype == torch.float32
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
    assert rel(gw, hw) <= 2.0 ** -15 and rel(gb, hb) <= 1e-5          # 64 tokens: dl in two bf16


@pytest.mark.parametrize("impl", ["torch", "cublaslt_nvfp4", "cublaslt_mxfp8"])
def test_training_step_with_every_option(impl):
    from backend import ops
    from models import TinyViT
    torch.manual_seed(0)
    m = TinyViT(**CFG, depth=2, linear_impl=impl, fused_norm=True, fuse_qkv=True, rope=True, qk_norm=True).cuda()
    x = torch.rand(64, 1, 28, 28, device="cuda")
    t = torch.randint(0, 10, (64,), device="cuda")
    before = dict(ops.LAUNCHES)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = m.loss(x, t)
    loss.backward()
    assert torch.isfinite(loss)
    for n, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), n
    assert ops.LAUNCHES["rotary"] - before["rotary"] == 2 * 3 and ops.LAUNCHES["xent"] > before["xent"]
    ops.check_status()


def test_training_script_replays_the_options_from_graphs():
    from backend import ops
    from train_tinyvit import train
    out = train("cublaslt_nvfp4", steps=3, warmup=1, batch=64, depth=2, seed=0, graph=True, fused_norm=True, fuse_qkv=True, rope=True,
                qk_norm=True, fused_loss=True)
    assert all(math.isfinite(v) for v in out["losses"]) and out["rope"] and out["qk_norm"] and out["fused_loss"]
    eager = train("cublaslt_nvfp4", steps=3, warmup=1, batch=64, depth=2, seed=0, rope=True, qk_norm=True, fused_loss=True)
    assert all(math.isfinite(v) for v in eager["losses"])
    ops.check_status()


def test_each_operator_differentiates_once():
    """A gradient taken with create_graph is there; a backward pass through it raises, as it does for torch's
    own functions that differentiate once."""
    from custom import FusedQKNorm, RotaryPositions, linear_cross_entropy
    rot = RotaryPositions(64, (32,)).cuda()
    norm = FusedQKNorm(64, rotary=rot).cuda()
    p = torch.arange(5, device="cuda")
    q = torch.randn(1, 5, 2, 64, device="cuda", requires_grad=True)
    h = torch.randn(8, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(30, 64, device="cuda").bfloat16().requires_grad_()
    t = torch.arange(8, device="cuda")
    for f, leaf in ((lambda: rot(q, positions=p).square().sum(), q), (lambda: norm(q, q, p)[0].square().sum(), q),
                    (lambda: linear_cross_entropy(h, w, t).square(), h)):
        (plain,) = torch.autograd.grad(f(), leaf)
        (g,) = torch.autograd.grad(f(), leaf, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="differentiates once"):
            g.float().square().sum().backward()


def test_partial_gradients_and_unused_outputs():
    """Only some inputs need gradients; only one of two outputs is used."""
    from custom import FusedQKNorm, RotaryPositions, linear_cross_entropy
    rot = RotaryPositions(64, (32,)).cuda()
    norm = FusedQKNorm(64, rotary=rot).cuda()
    p = torch.arange(5, device="cuda")
    q = torch.randn(1, 5, 2, 64, device="cuda", requires_grad=True)
    k = torch.randn(1, 5, 1, 64, device="cuda")
    a, b = rot(q, k, positions=p)
    assert a.requires_grad
    (g,) = torch.autograd.grad(a.sum(), q)
    assert torch.equal(g, torch.autograd.grad(rot(q, positions=p).sum(), q)[0])
    k.requires_grad_()
    a, b = norm(q, k, p)
    gq, gk, gw = torch.autograd.grad(b.sum(), [q, k, norm.q_weight])
    assert (gq == 0).all() and (gw == 0).all() and (gk != 0).any()
    h = torch.randn(70, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(30, 64, device="cuda").bfloat16()
    t = torch.arange(70, device="cuda") % 30
    (gh,) = torch.autograd.grad(linear_cross_entropy(h, w, t), h)          # a frozen head
    w2 = w.clone().requires_grad_()
    both = torch.autograd.grad(linear_cross_entropy(h, w2, t), [h, w2])
    assert torch.equal(gh, both[0])
    (gw,) = torch.autograd.grad(linear_cross_entropy(h.detach(), w2, t), w2)
    assert torch.equal(gw, both[1])
    with torch.no_grad():
        assert not linear_cross_entropy(h, w2, t).requires_grad


def test_weights_of_other_dtypes():
    """bf16 parameters: computed in fp32, gradients in their dtype."""
    from custom import FusedQKNorm
    norm = FusedQKNorm(64).cuda().bfloat16()
    q = torch.randn(2, 9, 2, 64, device="cuda", requires_grad=True)
    a, b = norm(q, q)
    g = torch.autograd.grad(a.sum() + b.square().sum(), [q, norm.q_weight, norm.k_weight])
    assert g[1].dtype == torch.bfloat16 and g[0].dtype == torch.float32 and all(torch.isfinite(x).all() for x in g)


def test_parameters_accumulate_like_any_others():
    from custom import FusedQKNorm
    norm = FusedQKNorm(64).cuda()
    q = torch.randn(2, 9, 2, 64, device="cuda")
    for _ in range(2):
        a, b = norm(q, q)
        (a.square().sum() + b.sum()).backward()
    once = torch.autograd.grad((lambda o: o[0].square().sum() + o[1].sum())(norm(q, q)), [norm.q_weight, norm.k_weight])
    assert torch.allclose(norm.q_weight.grad, 2 * once[0]) and torch.allclose(norm.k_weight.grad, 2 * once[1])


def _leaves_and_calls():
    """(leaves, call) of each operator: the call returns the tensor to differentiate."""
    from custom import FusedQKNorm, RotaryPositions, linear_cross_entropy
    gen = torch.Generator(device="cuda").manual_seed(11)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16).requires_grad_()

    rot = RotaryPositions(64, (16, 16)).cuda()
    norm = FusedQKNorm(64, rotary=rot).cuda()
    pos = torch.randint(0, 50, (40, 2), device="cuda", generator=gen)
    q, k, x, h, w = rand(2, 40, 3, 64), rand(2, 40, 3, 64), rand(2, 40, 192), rand(100, 64), rand(300, 64)
    t = torch.randint(0, 300, (100,), device="cuda", generator=gen)
    return {
        "rotary": ([q], lambda: rot(q, positions=pos)),
        "norm": ([q, k, norm.q_weight], lambda: torch.cat(norm(q, k, pos))),
        "norm_of_a_view": ([x], lambda: norm(x.view(2, 40, 3, 64), k.detach(), pos)[0]),
        "loss": ([h, w], lambda: linear_cross_entropy(h, w, t)),
    }


@pytest.mark.parametrize("which", ["rotary", "norm", "norm_of_a_view", "loss"])
def test_captured_backward_of_leaves_that_an_eager_graph_holds(which):
    """While an eager graph of the same leaves lives on the default stream the captured backward is refused, before
    anything that would spoil the capture; when it is gone the same call is captured and replays."""
    leaves, call = _leaves_and_calls()[which]
    eager = call()
    seed = torch.ones_like(eager)
    want = torch.autograd.grad(eager, leaves, seed, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
        with pytest.raises(RuntimeError, match="an eager graph of the same leaves"):
            torch.autograd.grad(out, leaves, seed)
    del out, graph
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, leaves, seed), want))
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaves, seed)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
