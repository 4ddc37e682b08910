"""Linear cross entropy: what needs no GPU (refusals, argument checks and workspace sizes of the C entries)."""
import pytest
import torch

from custom import LinearCrossEntropy, linear_cross_entropy


def test_refusals():
    h, w, t = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(10, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        linear_cross_entropy(h, w, t)
    for args in ((h, w, t[:3]), (h, w[0], t), (h[0], w, t)):
        with pytest.raises(ValueError, match=r"\(1 dimensions\)"):       # (numbers formatted in the native module)
            linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        linear_cross_entropy(h.float(), w, t)
    with pytest.raises(ValueError):
        LinearCrossEntropy(reduction="median")


def test_argument_errors_of_the_c_entries():
    from backend import _lib
    L = _lib.lib()
    buf = 0x10000

    def fwd(h=buf, ldh=64, w=buf, ldw=64, bias=None, bd=0, target=buf, T=4, D=64, V=10, red=1, loss=buf, ws=buf, n=1 << 30):
        return L.fp4t_linear_xent_forward(h, ldh, w, ldw, bias, bd, target, T, D, V, -100, red, loss, buf, buf, ws, n, None, None)

    def bwd(h=buf, ldh=64, T=4, D=64, V=10, red=1, dh=buf, dt=0, grad=buf, n=1 << 40):
        return L.fp4t_linear_xent_backward(grad, h, ldh, buf, 64, None, 0, buf, buf, T, D, V, -100, red, dh, dt, None, 0, None, 0,
                                           buf, n, None, None)

    for kw, word in ((dict(T=-1), "shape"), (dict(T=0), "tokens"), (dict(V=0), "shape"), (dict(D=60, ldh=64), "multiple of 8"), (dict(D=0), "shape"),
                     (dict(h=None), "null"), (dict(target=None), "null"), (dict(loss=None), "null"), (dict(ws=None), "null"),
                     (dict(ldh=56), "pitches"), (dict(ldw=68), "pitches"), (dict(h=buf + 8), "16-byte"), (dict(bias=buf + 4), "16-byte"),
                     (dict(bias=buf, bd=5), "bias"), (dict(target=buf + 4), "misaligned"), (dict(red=3), "reduction"), (dict(n=64), "workspace"),
                     (dict(T=2 ** 27), "shape"), (dict(T=2 ** 26, V=2 ** 26), "tiles")):
        assert fwd(**kw) == -1, kw
        assert word in L.fp4t_last_error().decode(), kw
    for kw, word in ((dict(T=0), "tokens"), (dict(D=63), "multiple of 8"), (dict(h=None), "null"), (dict(grad=None), "null"), (dict(dt=9), "gradients"),
                     (dict(dh=buf + 8), "16-byte"), (dict(red=-1), "reduction")):
        assert bwd(**kw) == -1, kw
        assert word in L.fp4t_last_error().decode(), kw
    assert bwd(dh=None) == 0                                    # nothing wanted, nothing launched
    size = L.fp4t_linear_xent_forward_workspace_bytes
    assert size(0, 8, 10) == 128 and size(-1, 8, 10) == -1 and size(10, 8, 0) == -1 and size(10, 9, 10) == -1
    # at most 16384 tokens' partial statistics at once (two numbers per 128 entries), and the packed rows
    assert size(10 ** 6, 64, 131072) < 1024 * 16384 * 8 + 10 ** 6 * (128 + 16) + (1 << 22)
    assert size(1, 64, 131072) < 1 << 15
