"""Thin torch-tensor wrappers over the C ABI (device pointers + current stream; no torch types cross the ABI)."""
from __future__ import annotations

import contextlib
import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .decoder import DecoderWeights

TQ = 64
POSE_PAD = 8


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def decode_batch(dec: DecoderWeights, latent: torch.Tensor, pts4: torch.Tensor, n_q: torch.Tensor,
                 mode: int = 0, pose_dim: int = 0):
    """latent (B,L) f32 cuda; pts4 (B,n_stride,4) f32 cuda (object frame); n_q (B,) int32 cuda.
    Returns y (B,n_stride) and, for mode 1, J (B,n_stride,L+8) rows [d/dz | pose-or-xyz | pad]."""
    assert latent.is_cuda and latent.dtype == torch.float32 and latent.is_contiguous()
    assert pts4.is_cuda and pts4.dtype == torch.float32 and pts4.is_contiguous() and pts4.shape[-1] == 4
    assert n_q.is_cuda and n_q.dtype == torch.int32
    B, n_stride = pts4.shape[0], pts4.shape[1]
    L = dec.latent_dim
    assert n_stride % TQ == 0 and latent.shape == (B, L)
    cb = torch.empty(2, B, 512, device=latent.device, dtype=torch.float32)
    y = torch.zeros(B, n_stride, device=latent.device, dtype=torch.float32)
    ldJ = L + POSE_PAD
    J = torch.zeros(B, n_stride, ldJ, device=latent.device, dtype=torch.float32) if mode == 1 else None
    rc = _lib.lib().hm_decode_batch(dec.handle, B, _ptr(latent), L, _ptr(pts4), _ptr(n_q), n_stride, _ptr(cb),
                                    _ptr(y), _ptr(J), ldJ, pose_dim, mode, _stream())
    _lib.check(rc, "hm_decode_batch")
    return y, J


# ---- training and adapting decoders

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # HM_TYPE_* of include/hortimapping_amd.h


def _rows(name: str, t: torch.Tensor) -> tuple:
    """(rows, columns, row stride) of a tensor whose last dimension is contiguous and whose other dimensions step as one."""
    if t.dim() == 0:
        raise ValueError(f"{name}: a scalar has no rows")
    cols = t.shape[-1]
    if t.numel() == 0:
        return t.numel() if cols == 0 else 0, cols, cols
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous, strides are {t.stride()} (call .contiguous())")
    rows, ld = 1, None                                   # innermost leading dimension first
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if ld is None:
            ld = s
        elif s != ld * rows:
            raise ValueError(f"{name}: rows must be equally spaced, shape {tuple(t.shape)} has strides {t.stride()} "
                             "(call .contiguous())")
        rows *= n
    ld = cols if ld is None else ld
    if rows > 1 and ld < cols:
        raise ValueError(f"{name}: rows overlap, shape {tuple(t.shape)} has strides {t.stride()} (call .contiguous())")
    return rows, cols, ld


def _rows_of_grad(t: torch.Tensor) -> tuple:
    """An incoming gradient may have any strides (an expanded one, a transposed one): copied where rows do not fit."""
    try:
        return (t,) + _rows("grad", t)
    except ValueError:
        t = t.contiguous()
        return (t,) + _rows("grad", t)


def _check_float(name: str, t: torch.Tensor, like: torch.Tensor = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if t.dtype not in TYPES:
        raise ValueError(f"{name}: float32, float16 or bfloat16 expected, got {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {like.dtype} on {like.device}")


def _check_draws(p, seed, tag, row0, device) -> tuple:
    """(p, seed as a number, seed tensor or None, tag, row0)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    word = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a seed tensor holds one int64 on {device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
        seed, word = 0, seed
    elif not 0 <= int(seed) < 1 << 64:
        raise ValueError(f"seed must be in [0, 2^64), got {seed}")
    if not 0 <= int(tag) < 1 << 32:
        raise ValueError(f"tag must be in [0, 2^32), got {tag}")
    if not 0 <= int(row0) < 1 << 63:
        raise ValueError(f"row0 must be in [0, 2^63), got {row0}")
    return p, int(seed), word, int(tag), int(row0)


def _no_tangents(**tensors) -> None:
    """Refuses forward-mode derivatives.  A tensor with a tangent does not require a gradient, so a call would compute the value
    and lose the tangent without a word."""
    if forward_ad._current_level < 0:                    # outside of every dual_level: no tensor has one
        return
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} carries a forward-mode tangent, but there are gradients in reverse mode only")


_HERE = contextlib.nullcontext()


def _on(device):
    """The device of a call's tensors as the current one (left alone where it is), and its current stream."""
    here = torch.cuda.current_device() == device.index
    return _HERE if here else torch.cuda.device(device), torch._C._cuda_getCurrentRawStream(device.index)


def _of_one_stream(y, stream):
    """y, a result whose backward pass hands gradients to leaves.  A leaf's node belongs to the stream on which the oldest
    living graph of that leaf was made, and the backward pass waits across streams: within a capture that pulls the older stream
    into it, and the process ends when the capture does.  So a node keeps its stream, and a capture on another is refused."""
    for node, _ in y.grad_fn.next_functions:
        if hasattr(node, "variable") and node.metadata.setdefault("hortimapping_stream", stream) != stream \
                and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a graph of the same leaves made on another stream is alive: its backward pass cannot be captured beside "
                               "it (drop or detach the results of the earlier calls first)")
    return y


def _dropout_forward(x, relu, draws):
    p, seed, word, tag, row0 = draws
    rows, cols, ld = _rows("x", x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    guard, stream = _on(x.device)
    with guard:
        _lib.check(_lib.lib().hm_dropout(x.data_ptr(), ld, y.data_ptr(), cols, rows, cols, TYPES[x.dtype], int(relu), p, seed,
                                         _ptr(word), tag, row0, stream), "hm_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, relu, draws):
        y = _dropout_forward(x, relu, draws)
        p, seed, word, tag, row0 = draws
        ctx.relu, ctx.draws = relu, (p, seed, tag, row0)
        ctx.save_for_backward(y if relu else None, word)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        y, word = ctx.saved_tensors
        p, seed, tag, row0 = ctx.draws
        dy, rows, cols, ld = _rows_of_grad(dy)
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
        guard, stream = _on(dy.device)
        with guard:
            _lib.check(_lib.lib().hm_dropout_backward(dy.data_ptr(), ld, _ptr(y), cols, dx.data_ptr(), cols, rows, cols,
                                                      TYPES[dy.dtype], int(ctx.relu), p, seed, _ptr(word), tag, row0, stream),
                       "hm_dropout_backward")
        return dx, None, None


def dropout(x: torch.Tensor, p: float, seed, *, tag: int = 0, row0: int = 0, relu: bool = False) -> torch.Tensor:
    """Dropout behind a hidden layer in training (`deepsdf/networks/deep_sdf_decoder.py:96-104`), its mask never stored:
    `keep * act(x) / (1 - p)` with act = ReLU when `relu`, differentiable in x.

    x (..., C) float32 / float16 / bfloat16 on the GPU, last dimension contiguous, rows equally spaced.  The mask comes from the
    counter-based generator Philox4x32-10 (include/hortimapping_amd.h has the definition) and depends on (seed, tag, row,
    column) alone; p is taken to the nearest 2^-16.  `seed`: an int, or an int64 tensor of one element on x's device that is
    read when the kernel runs (change it between replays of a captured graph; not between a forward pass and its backward).
    `tag`: number of the layer, so that one seed a step is enough.  `row0`: number of x's first row, so that a shard or a
    chunk of a batch draws what the whole batch would.  A NaN that is dropped is dropped: the result there is 0.
    Gradients are those of reverse mode, once; an x with a forward-mode tangent is refused."""
    _check_float("x", x)
    _no_tangents(x=x)
    draws = _check_draws(p, seed, tag, row0, x.device)
    if torch.is_grad_enabled() and x.requires_grad:
        return _of_one_stream(_Dropout.apply(x, bool(relu), draws), torch._C._cuda_getCurrentRawStream(x.device.index))
    return _dropout_forward(x, bool(relu), draws)


def _adapter_args(x, weight, bias, A, B, scale, row_start, adapter, draws) -> _lib.HmAdapterArgs:
    p, seed, word, tag, row0 = draws
    rows, k, ld = _rows("x", x)
    na, n, r = B.shape
    return _lib.HmAdapterArgs(TYPES[x.dtype], k, n, r, na, adapter.numel(), tag, rows, x.data_ptr(), ld, weight.data_ptr(),
                              weight.stride(0), _ptr(bias), A.data_ptr(), B.data_ptr(), _ptr(scale), row_start.data_ptr(),
                              adapter.data_ptr(), p, seed, _ptr(word), row0)


def _adapter_forward(x, weight, bias, A, B, scale, row_start, adapter, draws):
    args = _adapter_args(x, weight, bias, A, B, scale, row_start, adapter, draws)
    n, f32 = weight.shape[0], torch.float32
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    t = torch.empty(args.rows, (args.rank + 7) // 8 * 8, dtype=f32, device=x.device)
    guard, stream = _on(x.device)
    with guard:
        _lib.check(_lib.lib().hm_adapter_linear(ctypes.byref(args), y.data_ptr(), n, t.data_ptr(), stream), "hm_adapter_linear")
    return y, t


class _AdapterLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, A, B, weight, bias, scale, row_start, adapter, draws):
        y, t = _adapter_forward(x, weight, bias, A, B, scale, row_start, adapter, draws)
        p, seed, word, tag, row0 = draws
        ctx.draws = p, seed, tag, row0
        ctx.save_for_backward(x, A, B, weight, scale, row_start, adapter, t, word)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, A, B, weight, scale, row_start, adapter, t, word = ctx.saved_tensors      # (hooks may have moved them meanwhile)
        p, seed, tag, row0 = ctx.draws
        args = _adapter_args(x, weight, None, A, B, scale, row_start, adapter, (p, seed, word, tag, row0))
        dy, _, _, ld = _rows_of_grad(dy)
        want_x, want_a, want_b = ctx.needs_input_grad[:3]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
        dA = torch.empty_like(A) if want_a else None
        dB = torch.empty_like(B) if want_b else None
        lib = _lib.lib()
        size = lib.hm_adapter_linear_backward_bytes(ctypes.byref(args))
        if size < 0:
            _lib.check(int(size), "hm_adapter_linear_backward_bytes")
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        guard, stream = _on(x.device)
        with guard:
            _lib.check(lib.hm_adapter_linear_backward(ctypes.byref(args), dy.data_ptr(), ld, t.data_ptr(), _ptr(dx), x.shape[-1],
                                                      _ptr(dA), _ptr(dB), ws.data_ptr(), size, stream),
                       "hm_adapter_linear_backward")
        return dx, dA, dB, None, None, None, None, None, None


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, A: torch.Tensor, B: torch.Tensor, row_start: torch.Tensor,
                   adapter: torch.Tensor, *, bias: torch.Tensor = None, scale: torch.Tensor = None, p: float = 0.0, seed=0,
                   tag: int = 0, row0: int = 0) -> torch.Tensor:
    """A shared, frozen projection with the low-rank adapter of each request beside it (many species or cultivars on ONE
    decoder): `x W^T + bias + scale[a] dropout(x) A[a]^T B[a]^T`, differentiable in x, A and B.

    x (..., K) rows of all requests one after the other; weight (N, K); A (adapters, r, K), B (adapters, N, r); bias (N,);
    all of one type (float32 / float16 / bfloat16) on one GPU.  scale (adapters,) float32, default 1.  Request q holds the
    rows row_start[q] .. row_start[q + 1] - 1 (int32, ascending, S + 1 of them) and uses adapter[q] (int32, S); a value
    outside 0 .. adapters - 1, and rows of no request, get the bare projection.  Both are read on the GPU, when the kernels
    run: a captured graph may be replayed with others.  (Before a capture with a backward pass, drop the results of eager
    calls with the same leaves: beside a living one the call is refused, which sees leaves that are handed to both calls
    themselves, not those behind another operation.)  p, seed, tag, row0: dropout on the adapters' input, the mask of
    `dropout(x, p, seed, tag=tag, row0=row0)`.  Ranks up to 256, K and N up to 65536.
    Gradients are those of reverse mode, once; tensors with a forward-mode tangent are refused."""
    _check_float("x", x)
    for name, t in (("weight", weight), ("A", A), ("B", B)) + ((("bias", bias),) if bias is not None else ()):
        _check_float(name, t, x)
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} does not fit the weight {tuple(weight.shape)}")
    n, k = weight.shape
    if k > 1 and weight.stride(1) != 1 or n > 1 and weight.stride(0) < k:
        raise ValueError(f"weight: rows must be contiguous, strides are {weight.stride()}")
    if A.dim() != 3 or B.dim() != 3 or A.shape[2] != k or tuple(B.shape) != (A.shape[0], n, A.shape[1]):
        raise ValueError(f"A {tuple(A.shape)} and B {tuple(B.shape)} are not (adapters, r, {k}) and (adapters, {n}, r)")
    if not A.is_contiguous() or not B.is_contiguous():
        raise ValueError("A and B must be contiguous")
    if bias is not None and (tuple(bias.shape) != (n,) or not bias.is_contiguous()):
        raise ValueError(f"bias {tuple(bias.shape)} must be ({n},) and contiguous")
    if scale is not None and (tuple(scale.shape) != (A.shape[0],) or scale.dtype != torch.float32 or scale.device != x.device
                              or not scale.is_contiguous()):
        raise ValueError(f"scale must be ({A.shape[0]},) float32 on {x.device} and contiguous")
    for name, t in (("row_start", row_start), ("adapter", adapter)):
        if t.dtype != torch.int32 or t.device != x.device or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be one-dimensional, contiguous int32 on {x.device}")
    if row_start.numel() != adapter.numel() + 1:
        raise ValueError(f"{adapter.numel()} requests need {adapter.numel() + 1} row starts, got {row_start.numel()}")
    _no_tangents(x=x, weight=weight, A=A, B=B, bias=bias, scale=scale)
    draws = _check_draws(p, seed, tag, row0, x.device)
    if torch.is_grad_enabled():
        for name, t in (("weight", weight), ("bias", bias), ("scale", scale)):
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} requires a gradient, but the shared projection is frozen: adapter_linear gives "
                                 "gradients of x, A and B (detach it)")
        if x.requires_grad or A.requires_grad or B.requires_grad:
            return _of_one_stream(_AdapterLinear.apply(x, A, B, weight, bias, scale, row_start, adapter, draws),
                                  torch._C._cuda_getCurrentRawStream(x.device.index))
    return _adapter_forward(x, weight, bias, A, B, scale, row_start, adapter, draws)[0]
