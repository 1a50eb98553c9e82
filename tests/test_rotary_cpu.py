"""Rotary positions and norms of queries and keys on the CPU: against the framework's other rotary
functions, gradients against differences, and refusals."""
import math

import pytest
import torch

from drivedit_b200.layers.rope import RoPE3D, apply_rope, compute_rope_freqs, rope_apply, rope_table, yarn_inv_freqs
from drivedit_b200.layers.rope_v2 import RoPEConfig, RoPELayerV2
from drivedit_b200.ops.rotary import LAYOUTS, qk_norm_rotary, rotary


def _table(n, pairs):
    return rope_table(torch.rand(n, pairs, dtype=torch.float64) * 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_are_the_frameworks(dtype):
    x = torch.randn(2, 12, 3, 64).to(dtype)
    tab = RoPE3D(64, 2, 3, 4).table(2, 1)
    assert torch.equal(rotary(x, tab), apply_rope(x, tab))
    assert torch.equal(rotary(x, tab, inverse=True), apply_rope(x, tab, inverse=True))
    sin, cos = tab[:, None, :, 1], tab[:, None, :, 0]
    assert torch.equal(rotary(x, tab, layout="split"), rope_apply(x.float(), sin, cos).to(dtype))
    assert torch.equal(rotary(x, tab, layout="half"), rope_apply(x.float(), sin, cos, interleaved=False).to(dtype))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("R", [2, 6, 10])
def test_gradients(layout, R):
    x = torch.randn(2, 5, 3, 10, dtype=torch.float64, requires_grad=True)
    k = torch.randn(2, 5, 1, 10, dtype=torch.float64, requires_grad=True)
    w = torch.rand(10, dtype=torch.float64, requires_grad=True)
    tab, pos = _table(9, R // 2), torch.randint(0, 9, (2, 5))
    assert torch.autograd.gradcheck(lambda x: rotary(x, tab, pos, layout=layout), x)
    assert torch.autograd.gradgradcheck(lambda x: rotary(x, tab, pos, layout=layout), x)
    assert torch.autograd.gradcheck(lambda *t: qk_norm_rotary(*t, tab, pos, layout=layout), (x, k, w, w.detach().clone().requires_grad_()))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_inverse_is_the_transposed(layout):
    x = torch.randn(3, 4, 2, 12, dtype=torch.float64)
    tab = _table(7, 4)
    y = rotary(x, tab, offset=2, layout=layout)
    # a rotation by float32 cosines and sines keeps a pair's length to 2^-24 a factor
    assert torch.allclose(rotary(y, tab, offset=2, layout=layout, inverse=True), x, atol=1e-6)


def test_positions():
    x = torch.randn(2, 4, 3, 16)
    tab = _table(20, 8)
    at = torch.tensor([[3, 4, 5, 6], [9, 10, 11, 12]])
    y = rotary(x, tab, at)
    assert torch.equal(y[0], rotary(x[0], tab, offset=3)) and torch.equal(y[1], rotary(x[1:], tab, offset=9)[0])
    assert torch.equal(y, rotary(x, tab, at.int()))
    assert torch.equal(rotary(x, tab, at[0]), rotary(x, tab, at[:1]))
    for z in (x[:, :0], x[:0], x[:, :, :0]):
        assert rotary(z, tab).shape == z.shape
    assert torch.equal(rotary(x, tab[:, :0].contiguous()), x)


def test_layer_tables():
    """The layers' long-context tables: what RoPELayerV2 applies, position by position."""
    for cfg in (RoPEConfig(dim=32, max_seq_len=64, use_half_precision=False),
                RoPEConfig(dim=32, max_seq_len=256, original_max_seq_len=64, yarn_enabled=True, use_half_precision=False),
                RoPEConfig(dim=32, max_seq_len=64, ntk_alpha=2.0, use_half_precision=False)):
        layer = RoPELayerV2(cfg)
        x = torch.randn(2, 50, 3, 32)
        assert torch.equal(rotary(x, layer.table(50), layout="split"), layer(x))
        assert torch.equal(rotary(x, layer.table(53), offset=3, layout="split"), layer(x, start_pos=3))
    inv, _ = yarn_inv_freqs(32, 256, 64)
    want = rope_table(torch.outer(torch.arange(256, dtype=torch.float64), inv))
    yarn = RoPELayerV2(RoPEConfig(dim=32, max_seq_len=256, original_max_seq_len=64, yarn_enabled=True, use_half_precision=False))
    assert torch.allclose(yarn.table(256), want, atol=2 ** -24)
    sin, cos = compute_rope_freqs(32, 64)
    assert torch.equal(RoPELayerV2(RoPEConfig(dim=32, max_seq_len=64)).table(10)[..., 0], cos[:10])


def test_norm():
    q, k = torch.randn(2, 6, 4, 32, dtype=torch.float64), torch.randn(2, 6, 2, 32, dtype=torch.float64)
    q[0, 0, 0] = 0
    wq = torch.rand(32, dtype=torch.float64)
    a, b = qk_norm_rotary(q, k, wq)
    want = q / torch.sqrt(q.square().mean(-1, keepdim=True) + 1e-6) * wq
    assert torch.allclose(a, want, atol=1e-12) and torch.allclose(b.square().mean(-1), torch.ones(()).double(), atol=1e-4)
    assert not a[0, 0, 0].any()
    tab = _table(6, 16)
    for x, y in zip((a, b), qk_norm_rotary(q, k, wq, None, tab, layout="half")):
        assert torch.equal(rotary(x, tab, layout="half"), y)


def test_inplace():
    q, k, tab = torch.randn(1, 3, 4, 8).bfloat16(), torch.randn(1, 3, 2, 8).bfloat16(), _table(3, 4)
    want = qk_norm_rotary(q, k, table=tab)
    got = qk_norm_rotary(q, k, table=tab, inplace=True)
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    x = torch.randn(1, 3, 4, 8)
    want = rotary(x, tab)
    assert rotary(x, tab, inplace=True) is x and torch.equal(x, want)


def refusals(dev):
    """(what is wrong, call) on a device."""
    x, q, k = (torch.randn(*s, device=dev) for s in ((2, 4, 3, 16), (2, 4, 4, 16), (2, 4, 2, 16)))
    tab = _table(8, 8).to(dev)
    w = torch.ones(16, device=dev)
    leaf = x.clone().requires_grad_()
    return [
        ("rank", lambda: rotary(x[0, 0], tab)), ("odd heads", lambda: rotary(x[..., :15], tab)),
        ("large heads", lambda: rotary(torch.zeros(1, 1, 1, 258, device=dev), tab)),
        ("whole numbers", lambda: rotary(x.long(), tab)), ("layout", lambda: rotary(x, tab, layout="halves")),
        ("table's rank", lambda: rotary(x, tab[0])), ("table's pairs", lambda: rotary(x[..., :14], tab)),
        ("table's type", lambda: rotary(x, tab.double())), ("table's order", lambda: rotary(x, tab.transpose(0, 1))),
        ("table's gradient", lambda: rotary(x, tab.clone().requires_grad_())),
        ("table's length", lambda: rotary(x, tab, offset=5)), ("offset", lambda: rotary(x, tab, offset=-1)),
        ("far offset", lambda: rotary(x, tab, offset=1 << 62)),
        ("positions and offset", lambda: rotary(x, tab, torch.arange(4, device=dev), offset=1)),
        ("positions' type", lambda: rotary(x, tab, torch.arange(4, device=dev).float())),
        ("positions' shape", lambda: rotary(x, tab, torch.arange(5, device=dev))),
        ("positions' batch", lambda: rotary(x, tab, torch.zeros(3, 4, dtype=torch.long, device=dev))),
        ("positions of packed heads", lambda: rotary(x[0], tab, torch.zeros(1, 4, dtype=torch.long, device=dev))),
        ("in place of a leaf", lambda: rotary(leaf, tab, inplace=True)),
        ("tokens differ", lambda: qk_norm_rotary(q, k[:, :3], table=tab)), ("heads' sizes differ", lambda: qk_norm_rotary(q, k[..., :8])),
        ("types differ", lambda: qk_norm_rotary(q, k.bfloat16())), ("eps", lambda: qk_norm_rotary(q, k, eps=0.0)),
        ("eps NaN", lambda: qk_norm_rotary(q, k, eps=math.nan)), ("weight", lambda: qk_norm_rotary(q, k, w[:8])),
        ("weight's type", lambda: qk_norm_rotary(q, k, w.long())), ("positions alone", lambda: qk_norm_rotary(q, k, positions=torch.arange(4, device=dev))),
        ("offset alone", lambda: qk_norm_rotary(q, k, offset=1)),
        ("in place of a leaf, norm", lambda: qk_norm_rotary(leaf, x, inplace=True)),
    ]


@pytest.mark.parametrize("i", range(29))
def test_refusals(i):
    cases = refusals("cpu")
    assert len(cases) == 29
    what, call = cases[i]
    with pytest.raises(ValueError):
        call()


def test_position_outside_the_table():
    x, tab = torch.randn(1, 4, 2, 16), _table(8, 8)
    for bad in (-1, 8):
        with pytest.raises(IndexError):
            rotary(x, tab, torch.tensor([0, 1, bad, 2]))
