"""Low-rank adapters of many requests beside a shared projection (hm_adapter_linear) against a 64-bit restatement.

Tolerance of a sum of n products held in 32 bits, in whatever order: (n + 8) steps of 2^-23 of the sum of the absolute values
(each addition off by at most one step of a partial sum no larger than that), and half a step of the type for the one rounding
at the end.  What stands between the two products of the adapters is a sum of its own (n counts both) and is split into a high
and a low 16-bit part: off by 2^-16 of itself (bf16: half a step of the low part, 2^-8 of 2^-8), of its share of the sum."""
import numpy as np
import pytest
import torch

import adapter_oracle as AO
from hortimapping_amd import _lib, ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


class Case:
    def __init__(self, rows, k, n, r, lengths, which, na, dtype, seed=0, bias=True, scale=True, start=0):
        self.rows, self.k, self.n, self.r, self.na, self.dtype = rows, k, n, r, na, dtype
        self.start = [start]
        for v in lengths:
            self.start.append(self.start[-1] + v)
        self.which = list(which)
        assert self.start[-1] <= rows and len(self.which) == len(lengths)
        self.x = normal((rows, k), dtype, seed).requires_grad_()
        self.W = normal((n, k), dtype, seed + 1, k ** -0.5)
        self.A = normal((na, r, k), dtype, seed + 2, k ** -0.5).requires_grad_()
        self.B = normal((na, n, r), dtype, seed + 3, 0.5 * r ** -0.5).requires_grad_()
        self.b = normal((n,), dtype, seed + 4) if bias else None
        self.scale = normal((na,), torch.float32, seed + 5).abs() + 0.3 if scale else None
        self.dy = normal((rows, n), dtype, seed + 6, 0.1)
        self.row_start = torch.tensor(self.start, dtype=torch.int32, device="cuda")
        self.adapter = torch.tensor(self.which, dtype=torch.int32, device="cuda")

    def call(self, **kw):
        return ops.adapter_linear(self.x, self.W, self.A, self.B, self.row_start, self.adapter, bias=self.b, scale=self.scale, **kw)

    def check(self, backward=True, p=0.0, seed=0, tag=0):
        y = self.call(p=p, seed=seed, tag=tag)
        got = [y]
        if backward:
            got += list(torch.autograd.grad(y, (self.x, self.A, self.B), self.dy))
        keep, up = AO.keep_mask(self.rows, self.k, p, seed, tag) if p > 0 else (None, 1.0)
        ra = AO.segment_of_rows(self.start, self.which, self.rows, self.na)
        ref = [AO.adapter_linear(self.x, self.W, self.b, self.A, self.B, self.scale, ra, keep, up, self.dy if backward else None, m)
               for m in (False, True)]
        want, size = ref if backward else ([ref[0]], [ref[1]])
        most = max([0] + [int((ra == i).sum()) for i in range(self.na)])
        split = 0.0 if self.dtype == torch.float32 else 2.0 ** -16
        f = torch.finfo(self.dtype)
        count = (self.k + 2 * self.r, self.n + 2 * self.r, most + self.n, most + self.k)
        for name, g, w, s, c in zip(("y", "dx", "dA", "dB"), got, want, size, count):
            assert g.dtype == self.dtype and tuple(g.shape) == tuple(w.shape), name
            err = (g.detach().double().cpu() - w).abs()
            tol = ((c + 8) * 2.0 ** -23 + split) * s + f.eps / 2 * w.abs() + f.smallest_normal * f.eps
            assert bool((err <= tol).all()), (name, float((err / tol).max()), float(err.max()))
        return got


# rows, K, N, rank, lengths, adapters used, adapters
LAYOUTS = {
    "one row": (1, 8, 8, 4, [1], [0], 1),
    "one value": (1, 1, 1, 1, [1], [0], 1),
    "single rows": (9, 512, 512, 8, [1] * 9, [3, 0, -1, 2, 2, 7, 1, 0, 3], 4),          # -1 and 7: no adapter
    "single rows odd": (40, 259, 253, 13, [1] * 40, [i % 5 for i in range(40)], 5),
    "few rows": (64, 70, 33, 5, [30, 0, 34], [1, 0, 0], 2),
    "one more": (65, 64, 128, 16, [65], [0], 1),
    "ragged": (300, 259, 130, 7, [5, 0, 100, 1, 64, 30], [2, 1, 0, -1, 2, 1], 3),       # rows behind the last request
    "short": (301, 130, 70, 33, [7] * 43, [i % 4 for i in range(43)], 4),
    "tile crossing": (520, 64, 256, 64, [127, 2, 130, 261], [0, 1, 2, 1], 3),
    "big rank": (150, 96, 140, 70, [70, 80], [1, 0], 2),
    "bigger rank": (140, 40, 48, 256, [140], [0], 1),
    "no adapter": (130, 64, 64, 8, [100], [-1], 2),
    "unused adapter": (200, 128, 96, 16, [200], [1], 3),
    "wide": (257, 1031, 515, 16, [129, 128], [0, 1], 2),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", sorted(LAYOUTS))
def test_forward_and_backward(name, dtype):
    c = Case(*LAYOUTS[name], dtype)
    c.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["single rows odd", "few rows", "ragged", "short", "tile crossing", "big rank", "wide"])
def test_with_dropout_on_the_input(name, dtype):
    c = Case(*LAYOUTS[name], dtype, seed=40)
    c.check(p=0.3, seed=(1 << 45) + 17, tag=2)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_bias_scale_or_first_rows(dtype):
    Case(150, 72, 65, 6, [20, 90], [1, 0], 2, dtype, bias=False, scale=False, start=11).check()
    Case(20, 72, 65, 6, [5, 3], [1, 0], 2, dtype, bias=False, scale=False, start=11).check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_sizes_of_the_decoder(dtype):
    """First layer, the layer before the skip connection, a hidden layer: a few thousand points of eight instances."""
    for k, n, r, p in ((259, 512, 8, 0.2), (512, 253, 16, 0.0), (512, 512, 4, 0.2)):
        Case(5000, k, n, r, [1000, 300, 0, 700, 1024, 512, 900, 500], [0, 1, 2, 3, 0, -1, 2, 1], 4, dtype, seed=k).check(p=p, seed=5)


def test_no_requests_and_no_rows():
    c = Case(70, 32, 48, 4, [], [], 2, torch.float32)
    y, dx, dA, dB = c.check()
    assert not dA.any() and not dB.any()
    x = torch.zeros(0, 32, device="cuda", requires_grad=True)
    y = ops.adapter_linear(x, c.W, c.A, c.B, c.row_start, c.adapter)
    assert y.shape == (0, 48)
    dx, dA = torch.autograd.grad(y.sum(), (x, c.A))
    assert dx.shape == (0, 32) and dA.shape == c.A.shape and not dA.any()
    none = [t.detach()[:0] for t in (c.A, c.B)]
    y = ops.adapter_linear(c.x.detach(), c.W, *none, c.row_start, c.adapter, bias=c.b)
    want = c.x.detach().double() @ c.W.double().t() + c.b.double()
    assert float((y.double() - want).abs().max()) < 40 * 2.0 ** -23 * 40


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,lengths", [(12, [1] * 12), (300, [100, 60, 140])])
def test_the_mask_is_that_of_dropout(dtype, rows, lengths):
    """adapter_linear(p) equals the bare projection of x plus the adapters on ops.dropout(x): with weights of zero and exact
    inputs (powers of two) bit for bit."""
    which = [i % 2 for i in range(len(lengths))]
    c = Case(rows, 64, 96, 4, lengths, which, 2, dtype)
    x = torch.sign(c.x.detach())
    A = torch.sign(c.A.detach()) * 0.25
    B = torch.sign(c.B.detach())
    zero = torch.zeros_like(c.W)
    got = ops.adapter_linear(x, zero, A, B, c.row_start, c.adapter, p=0.5, seed=77, tag=4)
    want = ops.adapter_linear(ops.dropout(x, 0.5, 77, tag=4), zero, A, B, c.row_start, c.adapter)
    assert torch.equal(got, want) and bool(got.any())


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Rows of a wider buffer at odd places, a weight that is a slice, leading dimensions, gradients of any strides."""
    c = Case(150, 67, 51, 5, [50, 100], [1, 0], 2, dtype)
    c.check()
    wide = torch.zeros(150, 97, dtype=dtype, device="cuda")
    wide[:, 3:70] = c.x.detach()
    ww = torch.zeros(51, 99, dtype=dtype, device="cuda")
    ww[:, 1:68] = c.W
    x = wide[:, 3:70].view(3, 50, 67).requires_grad_()
    y = ops.adapter_linear(x, ww[:, 1:68], c.A, c.B, c.row_start, c.adapter, bias=c.b, scale=c.scale)
    ref = c.call()
    assert y.shape == (3, 50, 51) and torch.equal(y.view(150, 51), ref)
    dy = c.dy[:1, :1].expand(150, 51)
    a = torch.autograd.grad(y, (x, c.A, c.B), dy.reshape(3, 50, 51), retain_graph=True)
    b = torch.autograd.grad(ref, (c.x, c.A, c.B), dy)
    assert torch.equal(a[0].view(150, 67), b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    t = normal((51, 150), dtype, 9).t()
    ref = c.call()
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(ref, (c.x, c.A, c.B), t, retain_graph=True),
                                                 torch.autograd.grad(ref, (c.x, c.A, c.B), t.contiguous())))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,lengths", [(16, [4, 4, 4, 4]), (40, [1] * 40), (400, [130, 20, 130, 120])])
def test_an_infinity_stays_in_its_request(dtype, rows, lengths):
    """A broken adapter and a broken row reach their own rows and nothing else."""
    which = [i % 3 for i in range(len(lengths))]
    c = Case(rows, 64, 96, 8, lengths, which, 3, dtype)
    clean = [v.clone() for v in c.check()]
    ra = torch.from_numpy(AO.segment_of_rows(c.start, c.which, rows, 3)).cuda()
    with torch.no_grad():
        c.A[1].fill_(float("nan"))
        c.B[1].fill_(float("inf"))
        c.x[0, 5] = float("inf")                       # request 0, adapter 0
    y = c.call()
    dx, dA, dB = torch.autograd.grad(y, (c.x, c.A, c.B), c.dy)
    fine = (ra != 1)
    fine[0] = False
    assert torch.equal(y[fine], clean[0][fine])
    assert bool((~torch.isfinite(y[ra == 1])).all())
    other = ra != 1                                    # dx does not see x
    assert torch.equal(dx[other], clean[1][other])
    assert torch.equal(dA[2], clean[2][2]) and torch.equal(dB[2], clean[3][2])
    assert bool(torch.isnan(dA[1]).any()) and bool((~torch.isfinite(dA[0][:, 5])).all())
    assert torch.equal(dA[0][:, :5], clean[2][0][:, :5]) and torch.equal(dA[0][:, 6:], clean[2][0][:, 6:])


@pytest.mark.parametrize("dtype", TYPES)
def test_no_request_sees_the_batch_around_it(dtype):
    """The rows of a request are the same bits whatever the other requests hold."""
    a = Case(700, 128, 160, 16, [200, 300, 200], [0, 1, 2], 3, dtype)
    y = a.call(p=0.25, seed=3).detach()
    with torch.no_grad():
        a.x[:200].mul_(2)
        a.x[500:].zero_()
    assert torch.equal(a.call(p=0.25, seed=3)[200:500], y[200:500])


@pytest.mark.parametrize("rows,lengths,na", [(3000, [300] * 10, 3), (2000, [2] * 1000, 5)])
def test_same_bits_every_time(rows, lengths, na):
    c = Case(rows, 96, 130, 16, lengths, [i % na for i in range(len(lengths))], na, torch.bfloat16)
    a, b = c.check(p=0.1, seed=9), c.check(p=0.1, seed=9)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_so_many_requests_that_partial_sums_would_not_fit():
    """20000 requests of one row: sums over rows without slots."""
    rows = 20000
    c = Case(rows, 512, 140, 16, [1] * rows, [i % 7 - 1 for i in range(rows)], 6, torch.float32)
    c.check()


@pytest.mark.parametrize("start", [[0, 50, 30, 100], [0, 90, 20, 100], [-5, 40, 200, 100], [100, 60, 20, 0], [0, 2 ** 31 - 1, -2 ** 31, 7]])
def test_row_starts_that_do_not_ascend_stay_in_bounds(start):
    """Values of the rows concerned are unspecified; the call returns, and the next one is right."""
    c = Case(100, 64, 64, 8, [40, 30, 30], [0, 1, 0], 2, torch.float32)
    rs = torch.tensor(start, dtype=torch.int32, device="cuda")
    for x in (c.x, c.x[:10].detach().requires_grad_()):
        y = ops.adapter_linear(x, c.W, c.A, c.B, rs, c.adapter, bias=c.b, scale=c.scale)
        torch.autograd.grad(y.sum(), (x, c.A, c.B))
    torch.cuda.synchronize()
    c.check()


def test_gradient_against_differences():
    """<gradient, direction> against a central difference of the outputs in 64 bits: the map is bilinear in (A, B) and linear in
    x, so a difference in one of them is exact up to the rounding of the outputs."""
    c = Case(90, 48, 40, 6, [30, 60], [1, 0], 2, torch.float32, seed=3)
    y = c.call(p=0.2, seed=8)
    grads = torch.autograd.grad(y, (c.x, c.A, c.B), c.dy)
    for leaf, g in zip((c.x, c.A, c.B), grads):
        d = torch.sign(normal(leaf.shape, torch.float32, 77))
        h, keep = 2.0 ** -4, leaf.detach().clone()
        with torch.no_grad():
            leaf.copy_(keep + h * d)
            up = c.call(p=0.2, seed=8).double()
            leaf.copy_(keep - h * d)
            down = c.call(p=0.2, seed=8).double()
            leaf.copy_(keep)
        diff = float((((up - down) / (2 * h)) * c.dy.double()).sum())
        # 3600 outputs below 40, each off by (48 + 2 * 6 + 8) 2^-23 of it in either call, weighted with |dy|, over 2 h
        tol = 2 * 68 * 2.0 ** -23 * 40 / (2 * h) * float(c.dy.double().abs().sum()) + 1e-5 * abs(diff)
        assert abs(float((g.double() * d.double()).sum()) - diff) <= tol


def test_graph_replays_with_other_requests_and_seeds():
    c = Case(260, 64, 96, 8, [100, 60, 100], [0, 1, 2], 3, torch.bfloat16)
    word = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        y = c.call(p=0.25, seed=word)
        return [y] + list(torch.autograd.grad(y, (c.x, c.A, c.B), c.dy))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed, start, which in ((1, [0, 100, 160, 260], [0, 1, 2]), (2, [0, 7, 7, 200], [2, 0, -1]), (1 << 50, [3, 130, 131, 260], [1, 1, 0]),
                               (1, [0, 100, 160, 260], [0, 1, 2])):
        word.fill_(seed)
        c.row_start.copy_(torch.tensor(start, dtype=torch.int32))
        c.adapter.copy_(torch.tensor(which, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))        # eager work between the replays


def test_two_streams_at_once():
    cs = [Case(3000, 256, 256, 16, [1000, 500, 1500], [0, 1, 2], 3, torch.bfloat16, seed=i) for i in range(2)]

    def step(c):
        y = c.call()
        return [y] + list(torch.autograd.grad(y, (c.x, c.A, c.B), c.dy))
    want = [step(c) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = []
    for _ in range(3):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(step(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_gradients_asked_for_alone():
    c = Case(300, 64, 96, 8, [100, 200], [0, 1], 2, torch.float32)
    full = c.check()[1:]
    for i in range(3):
        leaves = [c.x, c.A, c.B]
        for j, v in enumerate(leaves):
            v.requires_grad_(j == i)
        (g,) = torch.autograd.grad(c.call(), leaves[i], c.dy)
        assert torch.equal(g, full[i])
        for v in leaves:
            v.requires_grad_(True)


def test_refusals():
    c = Case(70, 32, 48, 4, [30, 40], [0, 1], 2, torch.float32)
    base = dict(x=c.x, weight=c.W, A=c.A, B=c.B, row_start=c.row_start, adapter=c.adapter, bias=c.b, scale=c.scale)
    W = c.W.clone().requires_grad_()
    bad = [dict(x=c.x.double()), dict(x=c.x[:, :31]), dict(x=c.x.half()), dict(x=c.x.detach().t().contiguous().t()),
           dict(weight=c.W.t()), dict(weight=W), dict(weight=c.W.half()), dict(A=c.A[:1]), dict(A=c.A.transpose(0, 1)), dict(B=c.B[:, :, :2]),
           dict(B=c.B.transpose(1, 2).contiguous().transpose(1, 2)), dict(bias=c.b[:3]), dict(bias=c.b.clone().requires_grad_()),
           dict(scale=c.scale.double()), dict(scale=c.scale.clone().requires_grad_()), dict(scale=c.scale[:1]), dict(row_start=c.row_start.long()),
           dict(row_start=c.row_start[:2]), dict(adapter=c.adapter.cpu()), dict(p=1.1), dict(p=float("nan")), dict(seed=-1), dict(seed=c.scale)]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.adapter_linear(**{**base, **kw})
    with torch.no_grad():                                                 # frozen or not does not matter without gradients
        ops.adapter_linear(**{**base, "weight": W})
    r = torch.zeros(2, 300, 32, device="cuda"), torch.zeros(2, 48, 300, device="cuda")
    from hortimapping_amd._lib import HortiHipError
    with pytest.raises(HortiHipError, match="rank 300"):
        ops.adapter_linear(**{**base, "A": r[0], "B": r[1]})


@pytest.fixture
def tile():
    yield _lib.lib().hm_debug_set_adapter_tile
    _lib.lib().hm_debug_set_adapter_tile(0)


@pytest.mark.parametrize("side", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", sorted(LAYOUTS))
def test_every_tile_on_every_layout(tile, name, dtype, side):
    tile(side)
    Case(*LAYOUTS[name], dtype, seed=9).check()


@pytest.mark.parametrize("side", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["ragged", "short", "tile crossing", "big rank", "wide"])
def test_every_tile_with_dropout(tile, name, dtype, side):
    tile(side)
    Case(*LAYOUTS[name], dtype, seed=10).check(p=0.3, seed=77, tag=2)


@pytest.mark.parametrize("side", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_every_tile_with_hundreds_of_requests(tile, dtype, side):
    tile(side)
    for n in (255, 256, 700):                             # around what the wide tiles keep at hand
        Case(3 * n + 5, 130, 72, 6, [i % 7 for i in range(n)], [i % 6 - 1 for i in range(n)], 5, dtype, seed=n).check()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_reduction_at_the_wide_tile(tile, dtype):
    tile(256)
    for k in list(range(64, 75)) + [127, 128, 129, 191, 255]:
        Case(70, k, 40, 9, [33, 30], [0, 1], 2, dtype, seed=k).check()


# the wide tile (a tile a workgroup, "odd outputs" two for some): rows, K, N, rank, lengths, adapters used, adapters
WIDE = {
    "whole tiles": (16384, 512, 512, 8, [2048] * 8, [0, 1, 2, 0, 1, 2, -1, 0], 3),
    "ragged": (20001, 512, 515, 16, [1, 4999, 0, 37, 5000, 963, 6000, 2501], [0, 1, 2, 3, -1, 2, 1, 0], 4),
    "odd reduction": (30000, 259, 512, 5, [10000, 7, 9000, 10900], [2, 0, 1, 2], 3),
    "short tail": (20000, 66, 512, 12, [9999, 9999], [1, 0], 2),
    "odd outputs": (70000, 130, 253, 16, [30000, 20000, 20000], [0, 1, 0], 2),
    "big rank": (16500, 256, 512, 70, [8000, 8500], [1, 0], 2),
    "rank 64": (16640, 192, 640, 64, [130] * 128, [i % 5 for i in range(128)], 5),
    "many requests": (20480, 128, 512, 4, [40] * 512, [i % 7 - 1 for i in range(512)], 6),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", sorted(WIDE))
def test_wide_tiles(tile, name, dtype):
    tile(256)
    Case(*WIDE[name], dtype, seed=5).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["whole tiles", "ragged", "odd outputs", "rank 64", "many requests"])
def test_wide_tiles_with_dropout(tile, name, dtype):
    tile(256)
    Case(*WIDE[name], dtype, seed=6).check(p=0.3, seed=(1 << 40) + 3, tag=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_tiles_keep_an_infinity_in_its_request(tile, dtype):
    tile(256)
    lengths = [4000, 2, 6000, 6382]
    c = Case(16384, 128, 512, 8, lengths, [0, 1, 2, 0], 3, dtype)
    clean = [v.detach().clone() for v in c.check()]
    ra = torch.from_numpy(AO.segment_of_rows(c.start, c.which, c.rows, 3)).cuda()
    with torch.no_grad():
        c.A[1].fill_(float("nan"))
        c.B[1].fill_(float("inf"))
        c.x[5000, 7] = float("nan")
    y = c.call()
    dx, dA, dB = torch.autograd.grad(y, (c.x, c.A, c.B), c.dy)
    fine = ra != 1
    assert torch.equal(dx[fine], clean[1][fine])
    fine[5000] = False
    assert torch.equal(y[fine], clean[0][fine]) and bool((~torch.isfinite(y[ra == 1])).all())
    assert torch.equal(dA[0], clean[2][0]) and torch.equal(dB[0], clean[3][0])


def test_wide_tiles_in_a_graph_and_on_two_streams(tile):
    tile(256)
    cs = [Case(*WIDE["ragged"], torch.bfloat16, seed=i) for i in range(2)]

    def step(c):
        y = c.call(p=0.1, seed=4)
        return [y] + list(torch.autograd.grad(y, (c.x, c.A, c.B), c.dy))
    want = [[v.detach() for v in step(c)] for c in cs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cs], []
    for _ in range(2):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(step(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
    del got
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(cs[0])
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(cs[0])))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [64, 65, 129, 256, 257])
def test_few_rows_and_one_more(rows, dtype):
    Case(rows, 384, 272, 16, [1] * (rows - 3), [i % 9 - 1 for i in range(rows - 3)], 8, dtype).check(backward=False)
    Case(rows, 131, 77, 3, [rows // 2, rows - rows // 2], [1, 0], 2, dtype).check(backward=False)


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    c = Case(300, 64, 48, 4, [100, 150], [0, 1], 2, torch.float32)
    y = c.call()
    z = ops.dropout(c.x, 0.2, 3)
    want = [v.detach() for v in torch.autograd.grad(y, (c.x, c.A, c.B), c.dy, retain_graph=True)]
    torch.cuda.synchronize()
    for call in (c.call, lambda: ops.dropout(c.x, 0.2, 3)):
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="another stream"):
            with torch.cuda.graph(g):
                call()
    del y, z
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = torch.autograd.grad(c.call(), (c.x, c.A, c.B), c.dy)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_saved_tensors_that_were_moved_away(dtype):
    c = Case(300, 72, 48, 5, [100, 150], [0, 1], 2, dtype)

    def run(hooks):
        with hooks:
            h = c.x * 1
            y = ops.dropout(ops.adapter_linear(h, c.W * 1, c.A, c.B, c.row_start + 0, c.adapter + 0, bias=c.b, scale=c.scale * 1, p=0.2, seed=3),
                            0.3, 5, relu=True)
            del h
        junk = [torch.full_like(c.x, float("nan")) for _ in range(4)]
        out = torch.autograd.grad(y, (c.x, c.A, c.B), c.dy)
        del junk
        return out
    import contextlib
    for a, b in zip(run(torch.autograd.graph.save_on_cpu()), run(contextlib.nullcontext())):
        assert torch.equal(a, b)


def tiles_of_workgroups(rows, n):
    """Columns at which the 256-wide tiles of each workgroup start, in their order (eight runs of tiles, one for each part of the
    chip; 32 workgroups take turns in a run; bands of eight tiles of rows)."""
    tm, tn = -(-rows // 256), -(-n // 256)
    each, extra = divmod(tm * tn, 8)
    out = []
    for b in range(min(tm * tn, 256)):
        part = b % 8
        first = part * each + min(part, extra)
        mine = range(first + b // 8, first + each + (part < extra), 32)
        out.append([t % (8 * tn) // min(8, tm - t // (8 * tn) * 8) * 256 for t in mine])
    return out


# rows, K, N: at least three tiles a workgroup, other columns from one to the next but one
MANY = {
    "few rows in the last tile": (16228, 64, 4096),       # 100: two of the four waves have nothing to store there
    "three tiles of columns": (65536, 64, 768),
    "six tiles of columns": (24676, 64, 1536),
    "odd": (20060, 70, 2100),                             # 92 rows and 52 outputs in the last tiles, a tail of the reduction
    "half a tile of rows": (33000, 96, 1300),             # 232 rows in the last tiles
}


@pytest.mark.parametrize("adapters", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", sorted(MANY))
def test_many_tiles_a_workgroup(tile, name, dtype, adapters):
    """Tiles that one workgroup takes one after the other, with a bias that no two blocks of 64 outputs share: in 64 bits on the GPU."""
    rows, k, n = MANY[name]
    cols = tiles_of_workgroups(rows, n)
    assert sum(map(len, cols)) == -(-rows // 256) * -(-n // 256)
    assert any(len(c) >= 3 and c[i] != c[i + 2] for c in cols for i in range(len(c) - 2))
    # requests that end in one half of a tile's rows and not in the other, in the last rows too
    cuts = sorted({0, *range(300, rows, 1111), rows - 40, rows - 3}) if adapters else []
    lengths = [b - a for a, b in zip(cuts, cuts[1:])]
    c = Case(rows, k, n, 8, lengths, [i % 4 - 1 for i in range(len(lengths))], 3, dtype, seed=11)
    c.b = (torch.arange(n, device="cuda") // 64 * 3 - 90).to(dtype)      # whole numbers below 256: exact in every type
    tile(256)
    with torch.no_grad():
        y = c.call()
        ra = torch.from_numpy(AO.segment_of_rows(c.start, c.which, rows, 3)).cuda()
        sums = []
        for f in (lambda v: v.detach().double(), lambda v: v.detach().double().abs()):
            x, out = f(c.x), f(c.x) @ f(c.W).t() + f(c.b)
            for i in range(3):
                m = torch.nonzero(ra == i)[:, 0]
                out[m] += (x[m] @ f(c.A[i]).t() * f(c.scale[i])) @ f(c.B[i]).t()
            sums.append(out)
        want, size = sums
        f = torch.finfo(dtype)
        split = 0.0 if dtype == torch.float32 else 2.0 ** -16
        tol = ((k + 2 * 8 + 8) * 2.0 ** -23 + split) * size + f.eps / 2 * want.abs() + f.smallest_normal * f.eps
        err = (y.double() - want).abs()
        assert bool((err <= tol).all()), (float((err / tol).max()), torch.nonzero(err > tol)[:4].tolist())
        for _ in range(3):
            assert torch.equal(c.call(), y)


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_many_tiles_a_workgroup(tile, dtype, p):
    """dx has the tiles here: 97 x 6 of them."""
    assert max(map(len, tiles_of_workgroups(24676, 1536))) == 3
    tile(256)
    Case(24676, 1536, 64, 8, [4000, 60, 7000, 1, 9000, 4600], [0, 1, -1, 2, 1, 0], 3, dtype, seed=12).check(p=p, seed=6, tag=3)


@pytest.mark.parametrize("name", ["x", "weight", "A", "B", "bias", "scale"])
def test_forward_mode_is_refused(name):
    """A tensor with a tangent requires no gradient; its tangent must not vanish."""
    import torch.autograd.forward_ad as fwd
    c = Case(70, 32, 48, 4, [30, 40], [0, 1], 2, torch.float32)
    args = dict(x=c.x.detach(), weight=c.W, A=c.A.detach(), B=c.B.detach(), row_start=c.row_start, adapter=c.adapter, bias=c.b, scale=c.scale)
    y = ops.adapter_linear(**args)
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(NotImplementedError, match=f"{name} carries"):
            ops.adapter_linear(**args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match=f"{name} carries"):
            ops.adapter_linear(**args)
        args[name] = fwd.unpack_dual(args[name]).primal
        assert torch.equal(ops.adapter_linear(**args), y)                    # within a level, without a tangent


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_single_rows_than_one_dimension_of_a_grid(dtype):
    """Single rows times ranks over 2^28: 2^24 workgroups of 256 threads, 2^32 threads along one dimension, are refused by a launch.
    y and dx in 64 bits on the GPU."""
    rows, k, n, r, na = (1 << 20) + 64, 8, 8, 256, 3
    c = Case(rows, k, n, r, [], [], na, dtype, seed=21)
    c.row_start = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    c.adapter = torch.arange(rows, dtype=torch.int32, device="cuda") % (na + 1) - 1
    for v in (c.A, c.B):
        v.requires_grad_(False)                        # (sums over a million requests of one row are another matter)
    y = c.call()
    (dx,) = torch.autograd.grad(y, c.x, c.dy)
    which = c.adapter.long()
    f = torch.finfo(dtype)
    split = 0.0 if dtype == torch.float32 else 2.0 ** -16
    out = {}
    for size in (False, True):
        d = (lambda v: v.detach().double().abs()) if size else (lambda v: v.detach().double())
        W, s = d(c.W), d(c.scale)
        low = torch.stack([torch.zeros_like(W)] + [s[i] * (d(c.B[i]) @ d(c.A[i])) for i in range(na)])      # (n, k) of each adapter
        full = (W + low)[which + 1]
        out[size] = ((full * d(c.x)[:, None, :]).sum(2) + d(c.b), (full * d(c.dy)[:, :, None]).sum(1))
    for got, want, size, count in zip((y, dx), out[False], out[True], (k + 2 * r, n + 2 * r)):
        tol = ((count + 8) * 2.0 ** -23 + split) * size + f.eps / 2 * want.abs() + f.smallest_normal * f.eps
        err = (got.detach().double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


def test_transposes_of_more_adapters_than_one_dimension_of_a_grid():
    """65535 adapters of 16384 columns: 65535 x 257 workgroups transpose A and B.  dx of the rows, in 64 bits on the GPU."""
    na, k, n, rows, dtype = 65535, 16384, 8, 24, torch.bfloat16
    c = Case(rows, k, n, 1, [1] * rows, [0, na - 1, -1] + [(i * 7919) % na for i in range(rows - 3)], 1, dtype, seed=22)
    g = torch.Generator(device="cuda").manual_seed(5)
    c.A = torch.empty(na, 1, k, dtype=dtype, device="cuda").normal_(generator=g).mul_(k ** -0.5)
    c.B = torch.empty(na, n, 1, dtype=dtype, device="cuda").normal_(generator=g)
    c.scale = None
    (dx,) = torch.autograd.grad(c.call(), c.x, c.dy)
    f = torch.finfo(dtype)
    out = {}
    for size in (False, True):
        d = (lambda v: v.detach().double().abs()) if size else (lambda v: v.detach().double())
        a = c.adapter.long().clamp_min(0)
        u = (d(c.dy) * d(c.B[a][:, :, 0])).sum(1, keepdim=True) * (c.adapter >= 0)[:, None]
        out[size] = d(c.dy) @ d(c.W) + u * d(c.A[a][:, 0])
    tol = ((n + 2 + 8) * 2.0 ** -23 + 2.0 ** -16) * out[True] + f.eps / 2 * out[False].abs() + f.smallest_normal * f.eps
    err = (dx.double() - out[False]).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("side", [64, 128, 256])
def test_every_tile_on_odd_strides(tile, side, dtype):
    """x, weight and dy that start between vectors and have odd row strides: the bits of contiguous ones."""
    tile(side)
    c = Case(700, 333, 270, 12, [100, 37, 400, 130], [0, 2, -1, 1], 3, dtype, seed=30)
    want = c.check(p=0.2, seed=8)

    def odd(t, before, behind):
        w = torch.full((t.shape[0], t.shape[1] + before + behind), float("nan"), dtype=dtype, device="cuda")
        w[:, before:before + t.shape[1]] = t.detach()
        return w[:, before:before + t.shape[1]]
    x, W = odd(c.x, 3, 5).requires_grad_(), odd(c.W, 1, 3)
    y = ops.adapter_linear(x, W, c.A, c.B, c.row_start, c.adapter, bias=c.b, scale=c.scale, p=0.2, seed=8)
    got = [y] + list(torch.autograd.grad(y, (x, c.A, c.B), odd(c.dy, 5, 2)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("side", [64, 128, 256])
def test_offsets_past_32_bits(tile, side):
    """y, and then x and dx, of more than 2^31 values: the last rows are what a call on them alone gives."""
    rows, last, dtype = 530000, 1000, torch.bfloat16
    assert rows * 4096 > 2 ** 31
    tile(side)
    for k, n in ((64, 4096), (4096, 64)):
        c = Case(last, k, n, 8, [400, 600], [0, 1], 2, dtype, seed=31)
        want = c.call(p=0.1, seed=3, row0=rows - last)
        want = [want] + list(torch.autograd.grad(want, c.x, c.dy))
        x = torch.zeros(rows, k, dtype=dtype, device="cuda")
        x[-last:] = c.x.detach()
        dy = torch.zeros(rows, n, dtype=dtype, device="cuda")
        dy[-last:] = c.dy
        c.row_start = torch.tensor([0, rows - last, rows - 600, rows], dtype=torch.int32, device="cuda")
        c.adapter = torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda")
        c.x = x.requires_grad_()
        whole = c.call(p=0.1, seed=3)
        assert torch.equal(whole[-last:], want[0]) and torch.equal(whole[:2000], c.b.expand(2000, n))
        (dx,) = torch.autograd.grad(whole, c.x, dy)
        assert torch.equal(dx[-last:], want[1]) and not dx[:2000].any()
        del x, dy, whole, dx, c
