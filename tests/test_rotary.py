"""Rotary positions and query / key norms: what needs no GPU (tables, refusals, argument checks of the C entries)."""
import ctypes
import math

import pytest
import torch

from custom import FusedQKNorm, RotaryPositions


def fractions(rot):
    return [(int(t) % 2 ** 64) / 2.0 ** 64 for t in rot.turns]


def test_tables():
    r = RotaryPositions(16, (3, 2, 1), order="cycled", spectrum="shared", base=100.0)
    assert r.axis.tolist() == [0, 1, 2, 0, 1, 0]
    assert fractions(r) == pytest.approx([100.0 ** (-p / 6) / (2 * math.pi) for p in range(6)], rel=1e-15)
    r = RotaryPositions(16, (3, 2), order="blocks", spectrum="axis", base=100.0)
    assert r.axis.tolist() == [0, 0, 0, 1, 1]
    assert fractions(r) == pytest.approx([100.0 ** -e / (2 * math.pi) for e in (0, 1 / 3, 2 / 3, 0, 1 / 2)], rel=1e-15)
    # whole turns fall away, a negative frequency is the complement
    r = RotaryPositions(8, 2, frequencies=[2 * math.pi * 3.25, -2 * math.pi * 0.25])
    assert fractions(r) == pytest.approx([0.25, 0.75], abs=1e-15)
    assert r.table[2:] == (1, False)


def test_constructor_refusals():
    for kw in (dict(head_dim=15, sections=(2,)), dict(head_dim=16, sections=(9,)), dict(head_dim=16, sections=()),
               dict(head_dim=16, sections=(4, 0)), dict(head_dim=514, sections=(4,)), dict(head_dim=16, sections=(4,), layout="x"),
               dict(head_dim=16, sections=(4,), base=0.0), dict(head_dim=16, sections=(4,), frequencies=[1.0]),
               dict(head_dim=16, sections=(1,), frequencies=[float("inf")]), dict(head_dim=16, sections=(4,), order="x"),
               dict(head_dim=16, sections=(4,), spectrum="x")):
        with pytest.raises(ValueError):
            RotaryPositions(**kw)
    with pytest.raises(ValueError):
        FusedQKNorm(32, rotary=RotaryPositions(16, (4,)))
    with pytest.raises(ValueError):
        FusedQKNorm(32, eps=-1.0)
    with pytest.raises(ValueError):
        FusedQKNorm(33)


def test_no_cpu_path():
    rot = RotaryPositions(16, (4, 4))
    x, p = torch.zeros(2, 3, 1, 16), torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        rot(x, positions=p)
    with pytest.raises(NotImplementedError):
        FusedQKNorm(16, rotary=rot)(x, x, p)


def test_argument_errors_of_the_c_entries():
    from backend import _lib
    L = _lib.lib()
    buf = 0x10000

    def heads(n=2, data=buf, h=3, st=(192, 192, 64)):
        return (ctypes.c_int64 * (5 * n))(*([data or 0, h, *st] * n))

    def rotary(turned=8, axes=2, positions=buf, turns=buf, axis=buf):
        r = _lib.Rotary()
        r.positions, r.positions_i64, r.axes, r.turned, r.turns, r.axis = positions, 1, axes, turned, turns, axis
        return r

    def call(x=None, y=None, count=2, dtype=_lib.DT_F32, B=1, T=1, D=64, r=None):
        return L.fp4t_rotary(x or heads(), y or heads(), count, dtype, B, T, D, ctypes.byref(r or rotary()), 0, None)

    for rc, word in ((call(count=3), b"count"), (call(dtype=7), b"dtype"), (call(D=63), b"head_dim"), (call(D=514), b"head_dim"),
                     (call(r=rotary(turned=33)), b"turning"), (call(r=rotary(turned=-1)), b"turning"), (call(r=rotary(axes=0)), b"null"),
                     (call(r=rotary(turns=None)), b"null"), (call(r=rotary(positions=buf + 4)), b"misaligned"),
                     (call(x=heads(data=None)), b"null"), (call(x=heads(data=buf + 2)), b"aligned"), (call(y=heads(h=4)), b"heads"),
                     (call(x=heads(h=0), y=heads(h=0)), b"heads"), (call(B=-1), b"shape"), (call(B=2 ** 40, T=2 ** 40), b"shape")):
        assert rc == -1, word
    assert call(B=0) == 0 and call(T=0) == 0                 # nothing to do, nothing launched
    assert L.fp4t_rotary(None, heads(), 1, 1, 1, 1, 64, ctypes.byref(rotary()), 0, None) == -1
    assert L.fp4t_rotary(heads(), heads(), 1, 1, 1, 1, 64, None, 0, None) == -1
    w = (ctypes.c_void_p * 2)(buf, buf)
    w1 = (ctypes.c_void_p * 2)(buf, buf + 4)
    r = ctypes.byref(rotary())
    assert L.fp4t_qk_norm_rotary_forward(heads(), w1, 1e-6, heads(), 2, 1, 1, 1, 64, r, None) == -1 and b"weights" in L.fp4t_last_error()
    assert L.fp4t_qk_norm_rotary_forward(heads(), w, -1.0, heads(), 2, 1, 1, 1, 64, r, None) == -1 and b"eps" in L.fp4t_last_error()
    back = L.fp4t_qk_norm_rotary_backward
    assert back(heads(), heads(), w, 1e-6, heads(), w, 2, 1, 1, 1, 64, r, buf, 511, None) == -1 and b"workspace" in L.fp4t_last_error()
    assert back(heads(), heads(), w, 1e-6, heads(), w, 2, 1, 1, 1, 64, r, None, 4096, None) == -1 and b"workspace" in L.fp4t_last_error()
    assert back(None, heads(), w, 1e-6, heads(), w, 2, 1, 1, 1, 64, r, buf, 4096, None) == -1


def test_model_options_without_a_gpu():
    """`rope` adds no parameters, `qk_norm` two vectors per block; the plain model's state dict is unchanged."""
    from models import TinyViT
    from models.transformer_block import AttentionBlock
    plain = TinyViT(embed_dim=64, num_heads=4, depth=2)
    rope = TinyViT(embed_dim=64, num_heads=4, depth=2, rope=True)
    assert list(plain.state_dict()) == list(rope.state_dict())
    pos = rope.encoder[0].attn.positions
    assert pos.shape == (17, 2) and pos[0].tolist() == [0, 0] and pos[1].tolist() == [1, 1] and pos[-1].tolist() == [4, 4]
    both = TinyViT(embed_dim=64, num_heads=4, depth=2, rope=True, qk_norm=True)
    extra = set(both.state_dict()) - set(plain.state_dict())
    assert extra == {f"encoder.{i}.attn.qk_norm.{n}_weight" for i in (0, 1) for n in "qk"}
    assert both.encoder[0].attn.qk_norm.rotary is not None and both.encoder[0].attn.rotary is None
    with pytest.raises(ValueError):
        AttentionBlock(64, 4, rotary=RotaryPositions(16, (8,)))
    with pytest.raises(NotImplementedError):
        rope(torch.rand(2, 1, 28, 28))


def test_weights_and_tables_that_are_plain_attributes():
    """A parametrized or replicated module holds its weights and tables outside its parameter and buffer
    dictionaries: the call still finds them (and then refuses tensors that are not on a GPU)."""
    norm = FusedQKNorm(8, rotary=RotaryPositions(8, (2, 2)))
    q, pos = torch.zeros(3, 2, 8), torch.zeros(3, 2, dtype=torch.int64)

    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    torch.nn.utils.parametrize.register_parametrization(norm, "q_weight", Twice())
    with pytest.raises(NotImplementedError):
        norm(q, q, pos)
    replica = RotaryPositions(8, (2, 2))._replicate_for_data_parallel()
    replica._buffers = {}
    replica.turns, replica.axis = norm.rotary.turns, norm.rotary.axis
    assert replica.table[0] is norm.rotary.turns and replica.table[1:] == (norm.rotary.axis, 2, False)
