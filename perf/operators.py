"""What is measured of the operators around the quantized projections: rotary positions with
several axes, per-head query / key norms with that rotation in the same pass, and the softmax
cross entropy of a projection onto a large vocabulary.

Each case can be run in a plain form (elementary torch operations in 32 bits, rounded once at the
end) or, with `own = True`, through the package's public modules.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp4-training_b200")
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def _custom():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import custom
    return custom


# ------------------------------------------------------------------------------------- the cases
def _rot(name, op, batch, tokens, q_heads, k_heads, head_dim, sections, **more):
    c = {"name": name, "op": op, "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads,
         "head_dim": head_dim, "sections": sections, "base": 10000.0, "layout": "half", "order": "blocks",
         "spectrum": "axis", "dtype": "bf16", "train": False, "packed": True, "per_batch": False, "offset": 0}
    c.update(more)
    return c


def _xent(name, tokens, dim, vocab, **more):
    c = {"name": name, "op": "linear_cross_entropy", "tokens": tokens, "dim": dim, "vocab": vocab, "bias": False,
         "reduction": "mean", "ignored": 0.0, "train": True}
    c.update(more)
    return c


def listed():
    return [
        # one generated token of each of 16 requests, far into their contexts: latency
        _rot("rotary_decode", "rotary", 16, 1, 32, 8, 128, "64", offset=120000, per_batch=True),
        # a training step of the framework's own image model: 7 x 7 patches and a class token, rows and columns
        _rot("rotary_image_train", "rotary", 512, 50, 3, 3, 64, "16,16", base=100.0, train=True),
        # one long video sequence in training: time, height, width, grouped key heads
        _rot("rotary_video_train", "rotary", 1, 65536, 32, 8, 128, "16,24,24", spectrum="shared", base=1e6, train=True),
        # one token of one request: the smallest call
        _rot("qk_norm_decode", "qk_norm_rotary", 1, 1, 16, 8, 128, "64", base=1e6, offset=30000),
        # the image model's training step with normalised queries and keys
        _rot("qk_norm_image_train", "qk_norm_rotary", 512, 50, 3, 3, 64, "16,16", base=100.0, train=True),
        # long video sequences in training
        _rot("qk_norm_video_train", "qk_norm_rotary", 2, 16384, 32, 8, 128, "24,20,20", spectrum="shared", order="cycled",
             base=1e6, train=True),
        # a ragged shape: 32-bit tensors, adjacent pairs, a head of 80 of which 64 elements turn, an odd length
        _rot("qk_norm_ragged_fp32", "qk_norm_rotary", 3, 777, 5, 5, 80, "20,12", layout="interleaved", dtype="fp32", train=True,
             per_batch=True),
        # the framework's own classifier head: 512 images, 192 wide, 10 classes
        _xent("xent_classes", 512, 192, 10, bias=True),
        # the score of one token under a large vocabulary: the weight is read once
        _xent("xent_one_token", 1, 4096, 131072, train=False),
        # odd sizes, a bias, a third of the tokens padded out of the loss
        _xent("xent_odd", 2047, 1024, 50001, bias=True, ignored=0.33, reduction="sum"),
        # scoring: losses token by token, no gradient
        _xent("xent_scores", 4096, 768, 32768, reduction="none", train=False),
        # the largest: a training step of 8192 tokens, 4096 wide
        _xent("xent_large_train", 8192, 4096, 131072),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        tokens, dim, vocab = _log_int(rng, 1, 8192), 8 * _log_int(rng, 8, 512), _log_int(rng, 10, 131072)
        c = _xent("", tokens, dim, vocab, bias=rng.random() < 0.4, reduction=rng.choice(["mean", "sum", "none"]),
                  ignored=rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.9), 2)]), train=rng.random() < 0.7)
        del c["name"]
        return c
    axes = rng.choice([1, 2, 3])
    head_dim = 2 * _log_int(rng, 16, 128) if rng.random() < 0.3 else rng.choice([32, 48, 64, 80, 96, 128, 192, 256])
    pairs = head_dim // 2
    turned = pairs if rng.random() < 0.7 else rng.randint(max(axes, pairs // 4), pairs)
    cuts = sorted(rng.sample(range(1, turned), axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [turned])]
    k_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = k_heads * rng.choice([1, 1, 2, 4])
    rows = _log_int(rng, 1, 65536)                            # tokens over all sequences
    cap = 65536 * 40 * 128 // ((q_heads + k_heads) * head_dim)  # no larger than the largest listed case
    rows = max(1, min(rows, cap))
    batch = _log_int(rng, 1, min(rows, 512))
    c = _rot("", rng.choice(["rotary", "qk_norm_rotary"]), batch, max(1, rows // batch), q_heads, k_heads, head_dim,
             ",".join(str(s) for s in sections), base=rng.choice([100.0, 10000.0, 1e6]),
             layout=rng.choice(["half", "half", "interleaved"]), order=rng.choice(["blocks", "cycled"]),
             spectrum=rng.choice(["axis", "shared"]), dtype=rng.choice(["bf16", "bf16", "fp32"]), train=rng.random() < 0.7,
             packed=rng.random() < 0.7, per_batch=rng.random() < 0.5, offset=rng.choice([0, 0, _log_int(rng, 10, 1000000)]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------- inputs
def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _pair_table(case):
    """(axis, radians per position) of every turning pair."""
    sections = _sections(case)
    total = sum(sections)
    if case["order"] == "blocks":
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    else:                                   # round robin over the axes that have pairs left
        left, axis = list(sections), []
        while len(axis) < total:
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    axis.append(a)
    seen, freq = [0] * len(sections), []
    for p, a in enumerate(axis):
        e = seen[a] / sections[a] if case["spectrum"] == "axis" else p / total
        seen[a] += 1
        freq.append(case["base"] ** -e)
    return axis, freq


def _positions(case, gen, device):
    """[tokens, axes] or [batch, tokens, axes], int64: a text's index, an image's row and column
    behind a class token, or a video's frame, row and column."""
    tokens, axes = case["tokens"], len(_sections(case))
    i = torch.arange(tokens, device=device)
    if axes == 1:
        pos = i[:, None]
    elif axes == 2:
        side = max(1, math.isqrt(max(0, tokens - 1)))
        j = (i - 1).clamp_min(0)
        pos = torch.stack([j // side, j % side], dim=-1)
    else:
        side = max(1, round(tokens ** (1 / 3)))
        pos = torch.stack([i // (side * side), i // side % side, i % side], dim=-1)
    pos = pos + case["offset"]
    if case["per_batch"]:
        pos = pos[None] + torch.randint(0, 1000, (case["batch"], 1, 1), generator=gen, device=device)
    return pos


def _rot_inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    B, L, Hq, Hk, dh = (case[k] for k in ("batch", "tokens", "q_heads", "k_heads", "head_dim"))
    if case["packed"]:      # views of the stacked q / k / v projection's output
        x = torch.randn(B, L, (Hq + 2 * Hk) * dh, generator=gen, device=dev).to(dt)
        q = x[..., :Hq * dh].view(B, L, Hq, dh)
        k = x[..., Hq * dh:(Hq + Hk) * dh].view(B, L, Hk, dh)
    else:
        q = torch.randn(B, L, Hq, dh, generator=gen, device=dev).to(dt)
        k = torch.randn(B, L, Hk, dh, generator=gen, device=dev).to(dt)
    st = {"q": q, "k": k, "pos": _positions(case, gen, dev)}
    if case["op"] == "qk_norm_rotary":
        st["q_weight"] = 1.0 + 0.2 * torch.randn(dh, generator=gen, device=dev)
        st["k_weight"] = 1.0 + 0.2 * torch.randn(dh, generator=gen, device=dev)
    if case["train"]:       # gradients as an attention core returns them: head by head
        st["gq"] = torch.randn(B, Hq, L, dh, generator=gen, device=dev).to(dt).transpose(1, 2)
        st["gk"] = torch.randn(B, Hk, L, dh, generator=gen, device=dev).to(dt).transpose(1, 2)
    return st


def _xent_inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    T, D, V = case["tokens"], case["dim"], case["vocab"]
    std = 1.0 / math.sqrt(D)
    w = (torch.randn(V, D, generator=gen, device=dev) * std).to(torch.bfloat16)
    target = torch.randint(0, V, (T,), generator=gen, device=dev)
    h = torch.randn(T, D, generator=gen, device=dev)
    # half of the tokens are already predicted well: their state leans toward the target's row
    lean = 8.0 * torch.rand(T, 1, generator=gen, device=dev) * (torch.rand(T, 1, generator=gen, device=dev) < 0.5)
    h = (h + lean * w[target].float()).to(torch.bfloat16)
    ignore = torch.rand(T, generator=gen, device=dev) < case["ignored"]
    ignore[0] = False
    target = torch.where(ignore, torch.full_like(target, -100), target)
    st = {"h": h, "w": w, "target": target}
    if case["bias"]:
        st["b"] = (torch.randn(V, generator=gen, device=dev) * 0.1).to(torch.bfloat16)
    if case["train"]:
        st["g"] = torch.rand(T, generator=gen, device=dev) + 0.5 if case["reduction"] == "none" else torch.ones((), device=dev)
    return st


def prepare(case, seed):
    if case["op"] == "linear_cross_entropy":
        st = _xent_inputs(case, seed)
        if own:
            st["call"] = _custom().LinearCrossEntropy(ignore_index=-100, reduction=case["reduction"])
    else:
        st = _rot_inputs(case, seed)
        axis, freq = _pair_table(case)
        st["axis"] = torch.tensor(axis, device="cuda")
        st["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
        if own:
            c = _custom()
            rot = c.RotaryPositions(case["head_dim"], _sections(case), base=case["base"], layout=case["layout"],
                                    order=case["order"], spectrum=case["spectrum"])
            if case["op"] == "qk_norm_rotary":
                st["call"] = c.FusedQKNorm(case["head_dim"], rotary=rot, eps=EPS).cuda()
                with torch.no_grad():
                    st["call"].q_weight.copy_(st["q_weight"])
                    st["call"].k_weight.copy_(st["k_weight"])
            else:
                st["call"] = rot.cuda()
    st["case"] = dict(case)
    return st


# ------------------------------------------------------------------------------------- the plain form
def _split(x, n, layout):
    """The two members of every turning pair, and the elements behind them."""
    if layout == "half":
        return x[..., :n], x[..., n:2 * n], x[..., 2 * n:]
    return x[..., 0:2 * n:2], x[..., 1:2 * n:2], x[..., 2 * n:]


def _join(a, b, rest, layout):
    if layout == "half":
        return torch.cat([a, b, rest], dim=-1)
    return torch.cat([torch.stack([a, b], dim=-1).flatten(-2), rest], dim=-1)


def _turn(x, cos, sin, layout):
    a, b, rest = _split(x, cos.shape[-1], layout)
    return _join(a * cos - b * sin, a * sin + b * cos, rest, layout)


def _plain_rot(st):
    case = st["case"]
    layout, dt = case["layout"], _DTYPES[case["dtype"]]
    angle = st["pos"][..., st["axis"]].double() * st["freq"]     # far positions need 64 bits
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    out, grads, wgrads = [], [], []
    for name in ("q", "k"):
        x = st[name].float()
        if case["op"] == "qk_norm_rotary":
            w = st[name + "_weight"]
            r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
            xh = x * r
            out.append(_turn(xh * w, cos, sin, layout).to(dt))
        else:
            out.append(_turn(x, cos, sin, layout).to(dt))
        if case["train"]:
            g = _turn(st["g" + name].float(), cos, -sin, layout)
            if case["op"] == "qk_norm_rotary":
                wgrads.append((g * xh).sum((0, 1, 2)))
                u = g * w
                g = r * (u - xh * (u * xh).mean(-1, keepdim=True))
            grads.append(g.to(dt))
    return out + grads + wgrads


def _plain_xent(st):
    case = st["case"]
    h, w, target = st["h"].float(), st["w"].float(), st["target"]
    x = h @ w.T
    if case["bias"]:
        x = x + st["b"].float()
    keep = target != -100
    y = torch.where(keep, target, torch.zeros_like(target))[:, None]
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    s = e.sum(1, keepdim=True)
    loss = torch.where(keep, (s.log() + top - x.gather(1, y))[:, 0], torch.zeros((), device=x.device))
    count = keep.sum()
    out = {"mean": lambda: loss.sum() / count, "sum": loss.sum, "none": lambda: loss}[case["reduction"]]()
    if not case["train"]:
        return [out]
    g = st["g"] / count if case["reduction"] == "mean" else st["g"]
    g = torch.where(keep, g, torch.zeros((), device=x.device))[:, None]
    d = e / s
    d.scatter_add_(1, y, torch.full_like(g, -1.0))
    d = d * g
    res = [out, (d @ w).to(torch.bfloat16), (d.T @ h).to(torch.bfloat16)]
    if case["bias"]:
        res.append(d.sum(0).to(torch.bfloat16))
    return res


# ------------------------------------------------------------------------------------- the package's form
def _own_rot(st):
    case, call = st["case"], st["call"]
    if not case["train"]:
        with torch.no_grad():
            return list(call(st["q"], st["k"], positions=st["pos"]))
    q, k = st["q"].detach().requires_grad_(), st["k"].detach().requires_grad_()
    out = call(q, k, positions=st["pos"])
    leaves = [q, k] + ([call.q_weight, call.k_weight] if case["op"] == "qk_norm_rotary" else [])
    return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, [st["gq"], st["gk"]]))


def _own_xent(st):
    case = st["case"]
    b = st.get("b")
    if not case["train"]:
        with torch.no_grad():
            return [st["call"](st["h"], st["w"], st["target"], b)]
    leaves = [t.detach().requires_grad_() for t in (st["h"], st["w"], b) if t is not None]
    out = st["call"](leaves[0], leaves[1], st["target"], leaves[2] if b is not None else None)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, st["g"]))


def run(state):
    if state["case"]["op"] == "linear_cross_entropy":
        return _own_xent(state) if own else _plain_xent(state)
    return _own_rot(state) if own else _plain_rot(state)


# ------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["op"] == "linear_cross_entropy":
        T, D, V = case["tokens"], case["dim"], case["vocab"]
        nbytes = 2 * (T * D + V * D) + 8 * T + (2 * V if case["bias"] else 0)
        nbytes += 4 * T if case["reduction"] == "none" else 4
        flops = 2 * T * V * D
        if case["train"]:
            nbytes += 2 * (T * D + V * D) + (2 * V if case["bias"] else 0)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    es = 2 if case["dtype"] == "bf16" else 4
    rows = case["batch"] * case["tokens"]
    n = rows * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
    norm = case["op"] == "qk_norm_rotary"
    nbytes = 2 * n * es + 8 * len(_sections(case)) * (rows if case["per_batch"] else case["tokens"])
    flops = n * (6 if norm else 3)
    if case["train"]:
        nbytes += 2 * n * es        # the gradient read and written; the norm's input has been counted
        flops += n * (12 if norm else 3)
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_turn(x, angle, layout):
    n = angle.shape[-1]
    half = layout == "half"
    z = torch.complex(x[..., :n], x[..., n:2 * n]) if half else torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous())
    z = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[..., None, :])
    z = torch.cat([z[..., 0], z[..., 1]], dim=-1) if half else z.flatten(-2)
    return torch.cat([z, x[..., 2 * n:]], dim=-1)


def exact(case, seed):
    if case["op"] == "linear_cross_entropy":
        st = _xent_inputs(case, seed)
        leaves = [st[n].double().requires_grad_(case["train"]) for n in ("h", "w", "b") if n in st]
        x = torch.nn.functional.linear(leaves[0], leaves[1], leaves[2] if case["bias"] else None)
        keep = (st["target"] >= 0).nonzero()[:, 0]
        part = torch.logsumexp(x[keep], 1) - x[keep, st["target"][keep]]
        if case["reduction"] == "none":
            loss = torch.zeros(case["tokens"], dtype=torch.float64, device="cuda").index_put((keep,), part)
        else:
            loss = part.sum() if case["reduction"] == "sum" else part.mean()
        if not case["train"]:
            return [loss]
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves, st["g"].double()))
    st = _rot_inputs(case, seed)
    axis, freq = _pair_table(case)
    angle = torch.stack([st["pos"][..., a].double() * f for a, f in zip(axis, freq)], dim=-1)
    norm = case["op"] == "qk_norm_rotary"
    xs = [st[n].double().requires_grad_(case["train"]) for n in ("q", "k")]
    ws = [st[n + "_weight"].double().requires_grad_(case["train"]) for n in ("q", "k")] if norm else []
    ys = []
    for i, x in enumerate(xs):
        if norm:
            x = ws[i] * x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        ys.append(_exact_turn(x, angle, case["layout"]))
    if not case["train"]:
        return ys
    return [y.detach() for y in ys] + list(torch.autograd.grad(ys, xs + ws, [st["gq"].double(), st["gk"].double()]))
