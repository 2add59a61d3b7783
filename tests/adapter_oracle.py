"""Plain restatements in 64 bits of dropout and of low-rank adapters beside a projection (test infrastructure)."""
import numpy as np
import torch


def philox(counter, key):
    """Philox4x32-10 on arrays: counter (4, n), key two ints -> (4, n) uint64 holding 32-bit words."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(key[0]), int(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c)


def threshold(p):
    t = int(np.floor(p * 65536 + 0.5))
    return 65535 if t == 65536 and p < 1 else t


def keep_mask(rows, cols, p, seed, tag=0, row0=0):
    """((rows, cols) bool, factor) as include/hortimapping_amd.h defines them."""
    nb = -(-cols // 8)
    row = np.array([row0 + i for i in range(rows)], dtype=np.uint64)
    c = [np.tile(np.arange(nb, dtype=np.uint64), rows), np.repeat(row & np.uint64(0xFFFFFFFF), nb),
         np.repeat(row >> np.uint64(32), nb), np.full(rows * nb, tag, dtype=np.uint64)]
    w = philox(c, (seed % 2 ** 32, seed // 2 ** 32)) if rows * nb else np.zeros((4, 0), dtype=np.uint64)
    d = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], 1)          # (4, 2, n): low half first
    d = d.reshape(8, rows, nb).transpose(1, 2, 0).reshape(rows, nb * 8)[:, :cols]
    t = threshold(p)
    return torch.from_numpy(d >= t), (65536.0 / (65536 - t) if t < 65536 else 0.0)


def segment_of_rows(row_start, adapter, rows, n_adapters):
    """Adapter of every row, -1: none."""
    a = np.full(rows, -1, dtype=np.int64)
    for q, i in enumerate(adapter):
        if 0 <= i < n_adapters:
            a[row_start[q]:row_start[q + 1]] = i
    return a


def adapter_linear(x, W, b, A, B, scale, row_adapter, keep=None, up=1.0, dy=None, magnitude=False):
    """y, or (y, dx, dA, dB), in float64 on the CPU.  `magnitude`: the same sums over absolute values, what bounds the
    rounding of any order of summation."""
    f = (lambda v: v.detach().double().cpu().abs()) if magnitude else (lambda v: v.detach().double().cpu())
    x, W, A, B = f(x), f(W), f(A), f(B)
    s = f(scale) if scale is not None else torch.ones(A.shape[0], dtype=torch.float64)
    xd = x if keep is None else torch.where(keep, x * up, torch.zeros_like(x))
    y = x @ W.t() + (f(b) if b is not None else 0)
    out = [y]
    if dy is not None:
        dy = f(dy)
        dx, dA, dB = dy @ W, torch.zeros_like(A), torch.zeros_like(B)
        out += [dx, dA, dB]
    for i in range(A.shape[0]):
        m = torch.from_numpy(np.nonzero(row_adapter == i)[0])
        if m.numel() == 0:
            continue
        t = xd[m] @ A[i].t() * s[i]
        y[m] += t @ B[i].t()
        if dy is not None:
            u = dy[m] @ B[i] * s[i]
            dz = u @ A[i]
            dx[m] += dz if keep is None else torch.where(keep[m], dz * up, torch.zeros_like(dz))
            dA[i] += u.t() @ xd[m]
            dB[i] += dy[m].t() @ t
    return out[0] if dy is None else tuple(out)
