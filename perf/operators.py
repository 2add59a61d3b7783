"""Operators for training and adapting DeepSDF decoders: what is measured of them, and their plain forms.

`dropout`        y = keep * act(x) / (1 - p), keep drawn from the counter-based generator Philox4x32-10, never stored.
`adapter_linear` y = x W^T + b + s_a drop(x) A_a^T B_a^T: a shared projection with the low-rank adapter of each request
                 (an instance's points, a prompt, a single token) beside it; gradients of x, A and B.

The generator (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) has key (seed low, seed
high) and counter (column / 8, row low, row high, tag); its four 32-bit words are eight draws of 16 bits, low half first,
for the eight columns of the block.  A value is kept where its draw is at least round(65536 p), and p is the multiple of
1 / 65536 which that makes it."""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LOW = 0xFFFFFFFF


def listed():
    return [
        # latent dropout on the codes of one training batch of 64 shapes: a launch, and little else
        {"name": "drop codes f32", "op": "dropout", "rows": 64, "cols": 256, "type": "f32", "relu": False, "p": 0.2, "train": True},
        # a hidden layer of the 8 x 512 decoder, 64 shapes x 2048 samples: the training step's own size
        {"name": "drop hidden f32", "op": "dropout", "rows": 131072, "cols": 512, "type": "f32", "relu": True, "p": 0.2, "train": True},
        # the layer before the skip connection (512 - 256 - 3 outputs): odd rows, no vector of a row is aligned
        {"name": "drop skip bf16", "op": "dropout", "rows": 131072, "cols": 253, "type": "bf16", "relu": True, "p": 0.2, "train": True},
        # dropout kept on while decoding a voxel grid (spread of the sdf over masks): forward alone
        {"name": "drop grid f16", "op": "dropout", "rows": 32768, "cols": 512, "type": "f16", "relu": True, "p": 0.5, "train": False},
        # one point of each of 8 instances, an adapter each: latency
        {"name": "adapt points bf16", "op": "adapter", "requests": 8, "rows": 8, "k": 512, "n": 512, "adapters": 8, "rank": 8,
         "type": "bf16", "p": 0.0, "train": False},
        # 64 requests of one row each over a wide projection: the bytes of the weights
        {"name": "adapt tokens bf16", "op": "adapter", "requests": 64, "rows": 64, "k": 4096, "n": 4096, "adapters": 48, "rank": 16,
         "type": "bf16", "p": 0.0, "train": False},
        # prompts of unequal lengths
        {"name": "adapt ragged f16", "op": "adapter", "requests": 24, "rows": 6001, "k": 1024, "n": 4096, "adapters": 10, "rank": 32,
         "type": "f16", "p": 0.0, "train": False},
        # hidden layer, 64 instances x 1024 surface points, in the decoder's own type
        {"name": "adapt hidden f32", "op": "adapter", "requests": 64, "rows": 65536, "k": 512, "n": 512, "adapters": 6, "rank": 16,
         "type": "f32", "p": 0.0, "train": False},
        # the same layer in a training step of fewer shapes
        {"name": "adapt hidden f32 train", "op": "adapter", "requests": 16, "rows": 32768, "k": 512, "n": 512, "adapters": 6, "rank": 4,
         "type": "f32", "p": 0.0, "train": True},
        # first layer (256 codes + xyz in: odd rows), a whole training batch, with dropout on the adapters' input
        {"name": "adapt first bf16 train", "op": "adapter", "requests": 64, "rows": 131072, "k": 259, "n": 512, "adapters": 6, "rank": 8,
         "type": "bf16", "p": 0.2, "train": True},
        # the layer before the skip connection (odd outputs)
        {"name": "adapt skip f16 train", "op": "adapter", "requests": 64, "rows": 65536, "k": 512, "n": 253, "adapters": 64, "rank": 16,
         "type": "f16", "p": 0.0, "train": True},
        # wide layers: bound by the matrix products
        {"name": "adapt wide bf16 train", "op": "adapter", "requests": 16, "rows": 8192, "k": 4096, "n": 4096, "adapters": 16, "rank": 64,
         "type": "bf16", "p": 0.1, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("f32", "f16", "bf16"))
    train = rng.random() < 0.5
    if rng.random() < 0.35:
        cols = _log(rng, 1, 4096)
        return {"op": "dropout", "rows": _log(rng, 1, min(131072, 131072 * 512 // cols)), "cols": cols, "type": kind,
                "relu": rng.random() < 0.5, "p": rng.choice((0.05, 0.1, 0.2, 0.5, 0.77)), "train": train}
    k, n = (rng.choice((256, 512, 1024, 2048, 4096)) if rng.random() < 0.5 else _log(rng, 33, 4096) for _ in range(2))
    requests = _log(rng, 1, 256)
    most = min(131072, (8192 * 4096 * 4096 // (1 if kind != "f32" else 8)) // (k * n))
    rows = requests if not train and rng.random() < 0.4 else _log(rng, requests, max(requests, most))
    return {"op": "adapter", "requests": requests, "rows": rows, "k": k, "n": n, "adapters": _log(rng, 1, 64),
            "rank": rng.choice((1, 4, 8, 13, 16, 32, 64)), "type": kind, "p": rng.choice((0.0, 0.1)), "train": train}


def _lengths(case, seed):
    """Rows of each request: one each where there are as many rows as requests, else a random split (some may be empty)."""
    s, m = case["requests"], case["rows"]
    if s == m:
        return np.ones(s, dtype=np.int64)
    cuts = np.sort(np.random.RandomState(seed % (1 << 32)).randint(0, m + 1, s - 1))
    return np.diff(np.concatenate([[0], cuts, [m]]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = TYPES[case["type"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)
    m, train = case["rows"], case["train"]
    s = {"case": case, "seed": (int(seed) * 0x9E3779B97F4A7C15 + 12345) & ((1 << 63) - 1), "p": case["p"]}
    if case["op"] == "dropout":
        s["x"] = normal(m, case["cols"]).requires_grad_(train)
        if train:
            s["dy"] = normal(m, case["cols"], std=0.01)
        return s
    k, n, r, na = case["k"], case["n"], case["rank"], case["adapters"]
    rs = np.random.RandomState((int(seed) + 1) % (1 << 32))
    lengths = _lengths(case, int(seed))
    which = rs.randint(0, na, case["requests"])
    if case["requests"] >= 8:
        which[rs.randint(case["requests"])] = -1                     # a request without an adapter
    s["row_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()
    s["adapter"] = torch.from_numpy(which.astype(np.int32)).cuda()
    s["longest"] = int(lengths.max())
    s["x"] = normal(m, k).requires_grad_(train)
    s["W"] = normal(n, k, std=k ** -0.5)
    s["b"] = normal(n, std=0.1)
    s["A"] = normal(na, r, k, std=k ** -0.5).requires_grad_(train)
    s["B"] = normal(na, n, r, std=0.3 * r ** -0.5).requires_grad_(train)
    s["scale"] = torch.rand(na, generator=g, device="cuda") * 1.5 + 0.5
    if train:
        s["dy"] = normal(m, n, std=0.01)
    return s


def run(s):
    c = s["case"]
    if c["op"] == "dropout":
        return _dropout_own(s) if own else _dropout_plain(s)
    return _adapter_own(s) if own else _adapter_plain(s)


# ---- the framework's calls


def _dropout_own(s):
    from hortimapping_amd import ops
    y = ops.dropout(s["x"], s["p"], s["seed"], tag=3, relu=s["case"]["relu"])
    if not s["case"]["train"]:
        return {"y": y}
    (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y, "dx": dx}


def _adapter_own(s):
    from hortimapping_amd import ops
    y = ops.adapter_linear(s["x"], s["W"], s["A"], s["B"], s["row_start"], s["adapter"], bias=s["b"], scale=s["scale"],
                           p=s["p"], seed=s["seed"], tag=3)
    if not s["case"]["train"]:
        return {"y": y}
    dx, dA, dB = torch.autograd.grad(y, (s["x"], s["A"], s["B"]), s["dy"])
    return {"y": y, "dx": dx, "dA": dA, "dB": dB}


# ---- plain forms


def _wide_product(a, const):
    """High and low 32 bits of a 32-bit value (held in 64) times a 32-bit constant."""
    low = (a & 0xFFFF) * const
    high = (a >> 16) * const + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _keep_plain(rows, cols, p, seed, tag, device):
    """(rows, cols) truth values, and the factor of what is kept."""
    blocks = (cols + 7) // 8
    c0 = torch.arange(blocks, device=device, dtype=torch.int64).expand(rows, blocks)
    c1 = torch.arange(rows, device=device, dtype=torch.int64)[:, None].expand(rows, blocks)
    c2, c3 = torch.zeros_like(c1), torch.full_like(c1, tag)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):
        h0, l0 = _wide_product(c0, 0xD2511F53)
        h1, l1 = _wide_product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack([c0, c1, c2, c3], -1)
    draws = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, blocks * 8)[:, :cols]
    threshold = int(math.floor(p * 65536 + 0.5))
    return draws >= threshold, 65536.0 / (65536 - threshold)


def _dropout_plain(s):
    c, x = s["case"], s["x"].detach()
    keep, up = _keep_plain(c["rows"], c["cols"], s["p"], s["seed"], 3, x.device)
    v = x.float()
    if c["relu"]:
        keep = keep & (v > 0)
    y = torch.where(keep, v * up, 0.0).to(x.dtype)
    if not c["train"]:
        return {"y": y}
    return {"y": y, "dx": torch.where(keep, s["dy"].float() * up, 0.0).to(x.dtype)}


def _adapter_plain(s):
    c, dt = s["case"], s["x"].dtype
    m, k, n, r = c["rows"], c["k"], c["n"], c["rank"]
    x, W = s["x"].detach().float(), s["W"].float()
    # each request's rows as one matrix of a batch, padded to the longest
    row = torch.arange(m, device=x.device, dtype=torch.int32)
    seg = torch.searchsorted(s["row_start"], row, right=True) - 1
    pos = row - s["row_start"][seg]
    at = seg * s["longest"] + pos
    size = (c["requests"], s["longest"])
    a = s["adapter"].clamp_min(0).long()
    factor = torch.where(s["adapter"] >= 0, s["scale"][a], 0.0)[:, None, None]
    A, B = s["A"].detach()[a].float(), s["B"].detach()[a].float()
    xd, keep, up = x, None, 1.0
    if s["p"] > 0:
        keep, up = _keep_plain(m, k, s["p"], s["seed"], 3, x.device)
        xd = torch.where(keep, x * up, 0.0)
    xp = x.new_zeros(size[0] * size[1], k).index_copy_(0, at, xd).view(*size, k)
    t = torch.bmm(xp, A.transpose(1, 2)) * factor
    z = torch.bmm(t, B.transpose(1, 2)).view(-1, n)[at]
    y = (torch.addmm(s["b"].float(), x, W.t()) + z).to(dt)
    if not c["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dyp = x.new_zeros(size[0] * size[1], n).index_copy_(0, at, dy).view(*size, n)
    u = torch.bmm(dyp, B) * factor
    dz = torch.bmm(u, A).view(-1, k)[at]
    if keep is not None:
        dz = torch.where(keep, dz * up, 0.0)
    dx = (dy @ W + dz).to(dt)
    na = c["adapters"]
    dA = x.new_zeros(na, r, k).index_add_(0, a, torch.bmm(u.transpose(1, 2), xp)).to(dt)
    dB = x.new_zeros(na, n, r).index_add_(0, a, torch.bmm(dyp.transpose(1, 2), t)).to(dt)
    return {"y": y, "dx": dx, "dA": dA, "dB": dB}


# ---- from the definitions, in 64 bits


def _exact_keep(rows, cols, p, seed, tag):
    """The generator in unsigned 64-bit arithmetic on the host, a row of counters per eight columns."""
    nb = -(-cols // 8)
    c = np.zeros((4, rows * nb), dtype=np.uint64)
    c[0] = np.tile(np.arange(nb, dtype=np.uint64), rows)
    c[1] = np.repeat(np.arange(rows, dtype=np.uint64), nb)
    c[3] = tag
    key = [seed % 2 ** 32, seed // 2 ** 32]
    s32, low = np.uint64(32), np.uint64(LOW)
    for i in range(10):
        if i:
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(p1 >> s32) ^ c[1] ^ np.uint64(key[0]), p1 & low, (p0 >> s32) ^ c[3] ^ np.uint64(key[1]), p0 & low])
    w = np.ascontiguousarray(c.T).astype("<u4").view("<u2").reshape(rows, nb * 8)[:, :cols]
    drop = int(round(p * 65536))
    return torch.from_numpy(w >= drop).cuda().double() * (65536.0 / (65536 - drop))


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["op"] == "dropout":
        f = _exact_keep(case["rows"], case["cols"], case["p"], s["seed"], 3)
        if case["relu"]:
            f = f * (x > 0)
        return {"y": x * f, "dx": s["dy"].double() * f} if case["train"] else {"y": x * f}
    W, A, B = s["W"].double(), s["A"].detach().double(), s["B"].detach().double()
    f = _exact_keep(case["rows"], case["k"], case["p"], s["seed"], 3) if case["p"] > 0 else torch.ones_like(x)
    y = x @ W.t() + s["b"].double()
    out = {"y": y}
    if case["train"]:
        dy = s["dy"].double()
        dx, dA, dB = dy @ W, torch.zeros_like(A), torch.zeros_like(B)
        out.update(dx=dx, dA=dA, dB=dB)
    start, which, scale = s["row_start"].tolist(), s["adapter"].tolist(), s["scale"].double().tolist()
    for q, i in enumerate(which):
        if i < 0:
            continue
        at = slice(start[q], start[q + 1])
        t = (x[at] * f[at]) @ A[i].t() * scale[i]
        y[at] += t @ B[i].t()
        if case["train"]:
            u = dy[at] @ B[i] * scale[i]
            dx[at] += (u @ A[i]) * f[at]
            dA[i] += u.t() @ (x[at] * f[at])
            dB[i] += dy[at].t() @ t
    return out


def work(case):
    size = 4 if case["type"] == "f32" else 2
    m = case["rows"]
    if case["op"] == "dropout":
        e = m * case["cols"]
        return {"bytes": e * size * (4 if case["train"] else 2), "flops": e * (2 if case["train"] else 1)}
    k, n, r = case["k"], case["n"], case["rank"]
    used = min(case["requests"], case["adapters"])
    values = m * k + n * k + n + used * r * (k + n) + m * n
    flops = 2 * m * k * n + 2 * m * r * (k + n)
    if case["train"]:
        values += m * n + m * k + case["adapters"] * r * (k + n)
        flops += 2 * m * k * n + 4 * m * r * (k + n)
    return {"bytes": values * size, "flops": flops}
