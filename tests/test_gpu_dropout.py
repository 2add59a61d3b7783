"""Dropout (hm_dropout) against a 64-bit restatement of its definition; the mask bit for bit."""
import numpy as np
import pytest
import torch

import adapter_oracle as AO
from hortimapping_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1, 1), (1, 7), (3, 8), (5, 9), (64, 256), (33, 253), (1000, 15), (7, 4097), (2049, 1), (300, 512)]


def data(rows, cols, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + cols)
    return (torch.randn(rows, cols, generator=g, device="cuda") * std).to(dtype)


def close(got, want, dtype):
    """One product in 32 bits (its factor rounded to 32 bits) and one rounding to the type: half a step of each."""
    f = torch.finfo(dtype)
    rel = f.eps / 2 + 2 * 2.0 ** -24
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    err = (got - want).abs()
    assert bool((err <= rel * want.abs() + f.smallest_normal * f.eps / 2).all()), float(err.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("relu", [False, True])
def test_forward_and_backward(rows, cols, dtype, relu):
    x = data(rows, cols, dtype).requires_grad_()
    dy = data(rows, cols, dtype, 1, 0.01)
    seed, tag = 0x1234567890ABCDEF + rows, 9
    y = ops.dropout(x, 0.3, seed, tag=tag, relu=relu)
    (dx,) = torch.autograd.grad(y, x, dy)
    keep, up = AO.keep_mask(rows, cols, 0.3, seed, tag)
    xd = x.detach().double().cpu()
    if relu:
        keep = keep & (xd > 0)
    zero = torch.zeros_like(xd)
    close(y, torch.where(keep, xd * up, zero), dtype)
    close(dx, torch.where(keep, dy.double().cpu() * up, zero), dtype)
    assert torch.equal((y.detach() != 0).cpu(), keep & (xd != 0))          # the mask itself


@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 1e-6, 0.5, 0.77, 1 - 2.0 ** -18, 1.0])
@pytest.mark.parametrize("relu", [False, True])
def test_probabilities(p, relu):
    x = (data(65, 130, torch.float32).abs() + 0.1).requires_grad_()
    dy = data(65, 130, torch.float32, 2)
    y = ops.dropout(x, p, 3, relu=relu)
    (dx,) = torch.autograd.grad(y, x, dy)
    keep, up = AO.keep_mask(65, 130, p, 3)
    zero = torch.zeros(65, 130, dtype=torch.float64)
    close(y, torch.where(keep, x.detach().double().cpu() * up, zero), torch.float32)
    close(dx, torch.where(keep, dy.double().cpu() * up, zero), torch.float32)
    assert (p != 1.0) or not bool(y.any())
    assert (p != 0.0) or torch.equal(y, x)


def test_kept_share_and_independence():
    """A binomial share within six standard deviations; tags and seeds decide apart."""
    x = torch.ones(4096, 512, device="cuda")
    a, b, c = (ops.dropout(x, 0.2, s, tag=t) != 0 for s, t in ((1, 0), (1, 1), (2, 0)))
    n = x.numel()
    for m in (a, b, c):
        assert abs(float(m.double().mean()) - (1 - 13107 / 65536)) < 6 * (0.16 / n) ** 0.5
    for u, v in ((a, b), (a, c), (b, c)):
        assert abs(float((u & v).double().mean()) - (1 - 13107 / 65536) ** 2) < 6 * (0.25 / n) ** 0.5


def test_rows_of_a_shard_draw_what_the_batch_draws():
    x = data(100, 77, torch.bfloat16)
    y = ops.dropout(x, 0.4, 11, tag=2)
    assert torch.equal(ops.dropout(x[37:60], 0.4, 11, tag=2, row0=37), y[37:60])
    far = ops.dropout(x, 0.4, 11, tag=2, row0=(1 << 32) - 50)            # rows on both sides of 2^32
    keep, _ = AO.keep_mask(100, 77, 0.4, 11, 2, (1 << 32) - 50)
    assert torch.equal((far != 0).cpu(), keep & (x.cpu() != 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("relu", [False, True])
def test_strided_rows_and_shapes(dtype, relu):
    wide = data(40, 300, dtype)
    x = wide[:, 3:132].view(5, 8, 129)                                    # odd offset, row stride 300
    y = ops.dropout(x, 0.25, 5, relu=relu)
    assert y.shape == x.shape and y.is_contiguous()
    assert torch.equal(y.view(40, 129), ops.dropout(wide[:, 3:132].contiguous(), 0.25, 5, relu=relu))
    assert ops.dropout(wide[:0], 0.25, 5, relu=relu).shape == (0, 300)
    assert torch.equal(ops.dropout(wide[0], 0.25, 5), ops.dropout(wide[:1], 0.25, 5)[0])


def test_gradients_of_any_strides():
    x = data(64, 48, torch.float32).requires_grad_()
    y = ops.dropout(x, 0.5, 8)
    keep, up = AO.keep_mask(64, 48, 0.5, 8)
    for dy in (torch.ones((), device="cuda").expand(64, 48), data(48, 64, torch.float32).t(), data(64, 1, torch.float32).expand(64, 48)):
        (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
        close(dx, torch.where(keep, dy.double().cpu() * up, torch.zeros(64, 48, dtype=torch.float64)), torch.float32)


@pytest.mark.parametrize("relu", [False, True])
def test_infinities_and_nans(relu):
    x = data(50, 40, torch.float32)
    x[::3] = float("nan")
    x[1::3] = float("inf")
    y = ops.dropout(x, 0.5, 4, relu=relu)
    keep, _ = AO.keep_mask(50, 40, 0.5, 4)
    keep = keep.cuda()
    assert bool((y[~keep] == 0).all())                                    # what is dropped is 0
    assert bool(torch.isnan(y[::3][keep[::3]]).all()) and bool(torch.isinf(y[1::3][keep[1::3]]).all())


def test_gradient_against_differences():
    """The map is linear on either side of 0 for a fixed mask: a difference is exact up to the rounding of two products."""
    x = data(9, 21, torch.float32)
    x[x.abs() < 0.1] = 0.5
    x.requires_grad_()
    w = data(9, 21, torch.float32, 5)
    y = ops.dropout(x, 0.3, 6, relu=True)
    (dx,) = torch.autograd.grad(y, x, w)
    h = 2.0 ** -6
    with torch.no_grad():
        d = (ops.dropout(x + h, 0.3, 6, relu=True).double() - ops.dropout(x - h, 0.3, 6, relu=True).double()) / (2 * h)
    # two outputs up to 4 * 1.43, each off by 2^-23 of itself (x +- h rounded, the product rounded), over 2 h
    assert float((dx.double() - d * w.double()).abs().max()) <= 6 * 4 * 2.0 ** -23 * 2 / (2 * h) * float(w.abs().max())


def test_seed_tensor_and_graph_replays():
    x = data(200, 96, torch.float16).requires_grad_()
    dy = data(200, 96, torch.float16, 3)
    word = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        y = ops.dropout(x, 0.3, word, tag=1)
        return y, torch.autograd.grad(y, x, dy)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, dx = step()
    for seed in (5, 1 << 40, (1 << 63) - 1, 5):
        word.fill_(seed)
        g.replay()
        torch.cuda.synchronize()
        e = ops.dropout(x, 0.3, seed, tag=1)                              # eager work between the replays
        assert torch.equal(y, e)
        assert torch.equal(dx, torch.autograd.grad(e, x, dy)[0])


def test_other_streams():
    x = data(512, 512, torch.float32)
    want = ops.dropout(x, 0.5, 9, relu=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops.dropout(x, 0.5, 9, relu=True))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


def test_many_values():
    """More than 2^32 bytes: offsets past 32 bits; checked at the last rows."""
    rows, cols = (1 << 22) + 3, 515
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, 0.5, 21)
    keep, _ = AO.keep_mask(5, cols, 0.5, 21, 0, rows - 5)
    assert torch.equal((y[-5:] != 0).cpu(), keep)
    keep, _ = AO.keep_mask(5, cols, 0.5, 21)
    assert torch.equal((y[:5] != 0).cpu(), keep)


def test_refusals():
    x = data(8, 8, torch.float32)
    for bad in (x.double(), x.t(), x.expand(2, 8, 8), x[0, 0]):
        with pytest.raises(ValueError):
            ops.dropout(bad, 0.5, 1)
    for kw in (dict(p=1.5), dict(p=-1), dict(p=float("nan")), dict(seed=-1), dict(seed=1 << 64), dict(tag=1 << 32), dict(row0=-1),
               dict(seed=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(seed=torch.zeros(1, dtype=torch.int64)),
               dict(seed=torch.zeros(1, device="cuda"))):
        with pytest.raises(ValueError):
            ops.dropout(x, **{"p": 0.5, "seed": 1, **kw})


def test_a_seed_changed_before_the_backward_pass_is_an_error():
    x = data(8, 8, torch.float32).requires_grad_()
    word = torch.ones(1, dtype=torch.int64, device="cuda")
    y = ops.dropout(x, 0.5, word)
    word.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("relu", [False, True])
def test_forward_mode_is_refused(relu):
    """A tensor with a tangent requires no gradient; its tangent must not vanish."""
    import torch.autograd.forward_ad as fwd
    x = torch.randn(4, 9, device="cuda")
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="x carries"):
            ops.dropout(d, 0.3, 5, relu=relu)
        assert torch.equal(ops.dropout(fwd.unpack_dual(d).primal, 0.3, 5, relu=relu), ops.dropout(x, 0.3, 5, relu=relu))
    with pytest.raises(NotImplementedError, match="x carries"):
        torch.func.jvp(lambda t: ops.dropout(t, 0.3, 5, relu=relu), (x,), (x,))


@pytest.mark.parametrize("relu", [False, True])
def test_offsets_past_32_bits(relu):
    """More than 2^31 values: the last rows are what a call on them alone gives."""
    rows, cols, last = 530000, 4099, 300
    assert rows * 4096 > 2 ** 31
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-last:] = data(last, cols, torch.bfloat16)
    part = x[-last:].clone().requires_grad_()
    x.requires_grad_()
    y, z = ops.dropout(x, 0.3, 11, tag=2, relu=relu), ops.dropout(part, 0.3, 11, tag=2, row0=rows - last, relu=relu)
    assert torch.equal(y[-last:], z) and not y[:1000].any() and bool(z.any())
    dy = torch.ones_like(x)
    (dx,), (dz,) = torch.autograd.grad(y, x, dy), torch.autograd.grad(z, part, dy[-last:])
    assert torch.equal(dx[-last:], dz) and bool(dz.any())
