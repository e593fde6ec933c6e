"""Plain 64-bit NumPy forms of the operators for several element types, and how far a kernel may be from them."""
import numpy as np
import torch

# half a step of each type, relative to the value
HALF_STEP = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half a step of the smallest values
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
# what sums and statistics are held in
WIDE_HALF_STEP = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -24,
                  torch.bfloat16: 2.0 ** -24}


def host64(t):
    return t.detach().double().cpu().numpy()


# --------------------------------------------------------------------------- group normalisation
def _grouped(t, groups, nhwc):
    """(batch, ..., channels) or (batch, channels, ...) -> (batch, pixels, groups, channels of a group)"""
    n = t.shape[0]
    c = t.shape[-1] if nhwc else t.shape[1]
    t = t.reshape(n, -1, c) if nhwc else t.reshape(n, c, -1).transpose(0, 2, 1)
    return t.reshape(n, t.shape[1], groups, c // groups)


def _ungrouped(t, shape, nhwc):
    t = t.reshape(t.shape[0], t.shape[1], -1)
    return (t if nhwc else t.transpose(0, 2, 1)).reshape(shape)


def silu_derivative(z):
    p = 1 / (1 + np.exp(-z))
    return p * (1 + z * (1 - p))


def gn_forward(x, gamma, beta, groups, eps, activation, nhwc):
    xg = _grouped(x, groups, nhwc)
    mean = xg.mean(axis=(1, 3))
    var = ((xg - mean[:, None, :, None]) ** 2).mean(axis=(1, 3))
    inv_std = 1 / np.sqrt(var + eps)
    z = (xg - mean[:, None, :, None]) * inv_std[:, None, :, None] * gamma.reshape(groups, -1) + beta.reshape(groups, -1)
    y = np.where(z > 0, z, 0) if activation == "relu" else z / (1 + np.exp(-z)) if activation == "silu" else z
    return _ungrouped(y, x.shape, nhwc), mean, inv_std


def gn_forward_bounds(x, gamma, beta, groups, eps, nhwc, y, dtype):
    """How far (y, mean, inv_std) may be off.  A sum of n terms that are each rounded is off by about sqrt(n) half steps of
    the sum of magnitudes; 8 sqrt(n) + 8 is taken.  With R the largest distance of a group's element from its mean, the terms
    are at most 2 R and 4 R^2 (they are differences from an element)."""
    u, out = WIDE_HALF_STEP[dtype], HALF_STEP[dtype]
    xg = _grouped(x, groups, nhwc)
    n = xg.shape[1] * xg.shape[3]
    k = (8 * np.sqrt(n) + 8) * u
    mean = xg.mean(axis=(1, 3), keepdims=True)
    d = np.abs(xg - mean)
    r = d.max(axis=(1, 3), keepdims=True)
    var = (d ** 2).mean(axis=(1, 3), keepdims=True)
    d_mean = 2 * u * np.abs(mean) + 2 * k * r
    # the rounded mean of a piece enters the variance by its square
    d_var = 8 * k * r ** 2 + d_mean ** 2
    inv = 1 / np.sqrt(var + eps)
    rel = d_var / (2 * (var + eps)) + 2 * u
    g, b = np.abs(gamma).reshape(groups, -1), np.abs(beta).reshape(groups, -1)
    d_z = g * (d * inv * (rel + 4 * u) + inv * (1 + rel) * d_mean) + 2 * u * (g * d * inv + b)
    # the slope of an activation is at most 1.1; its own arithmetic is 8 half steps of z
    z = g * d * inv + b
    d_y = 1.1 * d_z + 8 * u * z
    return _ungrouped(d_y, x.shape, nhwc) + out * np.abs(y) + TINY[dtype], d_mean[:, 0, :, 0], (rel * inv)[:, 0, :, 0]


def gn_backward(dy, x, gamma, beta, mean, inv_std, groups, activation, nhwc):
    xg, dz = _grouped(x, groups, nhwc), _grouped(dy, groups, nhwc)
    g, b = gamma.reshape(groups, -1), beta.reshape(groups, -1)
    r = inv_std[:, None, :, None]
    xn = (xg - mean[:, None, :, None]) * r
    z = xn * g + b
    if activation == "relu":
        dz = dz * (z > 0)
    elif activation == "silu":
        dz = dz * silu_derivative(z)
    a = (dz * g).mean(axis=(1, 3), keepdims=True)
    bb = (dz * g * xn).mean(axis=(1, 3), keepdims=True)
    dx = r * (g * dz - a - xn * bb)
    return (dz * xn).sum(axis=(0, 1)).reshape(-1), dz.sum(axis=(0, 1)).reshape(-1), _ungrouped(dx, x.shape, nhwc)


def gn_backward_bounds(dy, x, gamma, beta, mean, inv_std, groups, activation, nhwc, dx, dtype):
    """How far (dgamma, dbeta, dx) may be off: sums as in ``gn_forward_bounds``; xn is off by 3 half steps, and silu's
    derivative by 0.5 (the largest of its second derivative) times z's error, 4 half steps of |gamma xn| + |beta|, and by
    8 (1 + |z|) half steps of its own arithmetic."""
    u, out = WIDE_HALF_STEP[dtype], HALF_STEP[dtype]
    xg, dyg = _grouped(x, groups, nhwc), np.abs(_grouped(dy, groups, nhwc))
    g, b = np.abs(gamma).reshape(groups, -1), np.abs(beta).reshape(groups, -1)
    r = inv_std[:, None, :, None]
    xn = np.abs((xg - mean[:, None, :, None]) * r)
    z = g * xn + b
    if activation == "silu":
        dz, d_dz = 1.1 * dyg, dyg * (0.5 * 4 * u * z + 8 * u * (1 + z))
    else:
        dz, d_dz = dyg, 0.0 * dyg
    n = xg.shape[1] * xg.shape[3]
    k, k_all = ((8 * np.sqrt(v) + 8) * u for v in (n, xg.shape[0] * xg.shape[1]))
    d_gamma = (k_all * dz * xn + d_dz * xn + 4 * u * dz * xn).sum(axis=(0, 1))
    d_beta = (k_all * dz + d_dz).sum(axis=(0, 1))

    def mean_of(v):
        return v.mean(axis=(1, 3), keepdims=True)

    a, bb = mean_of(g * dz), mean_of(g * dz * xn)
    d_a = (k + 4 * u) * a + mean_of(g * d_dz)
    d_b = (k + 8 * u) * bb + mean_of(g * d_dz * xn)
    d_dx = r * (g * d_dz + d_a + xn * d_b + 4 * u * (g * dz + a + xn * bb))
    return (d_gamma.reshape(-1), d_beta.reshape(-1),
            _ungrouped(d_dx, x.shape, nhwc) + out * np.abs(dx) + TINY[dtype])


# --------------------------------------------------------------------------- dropout
def philox4x32_10(counter, key):
    """``counter``: four arrays of 32-bit words, ``key``: two words; the four words of each call."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_numbers(first, count, seed, offset):
    """The 16-bit numbers of elements first .. first + count - 1; first is a multiple of 8."""
    call = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = philox4x32_10([call & low, call >> half, np.full_like(call, offset & 0xFFFFFFFF), np.full_like(call, offset >> 32)],
                      [seed & 0xFFFFFFFF, seed >> 32])
    u = np.stack([w >> s & np.uint64(0xFFFF) for w in c for s in (np.uint64(0), np.uint64(16))], axis=1)
    return u.reshape(-1)[:count].astype(np.int64)


def dropout(x, rate, seed, offset):
    """What the kernel has to return bit for bit: one product in 32 bits (64 for float64), rounded once to the type."""
    threshold = int(np.round(rate * 65536))
    keep = torch.from_numpy(dropout_numbers(0, x.numel(), seed, offset) >= threshold).view(x.shape)
    wide = x.cpu() if x.dtype == torch.float64 else x.cpu().float()
    scale = torch.tensor(65536 / (65536 - threshold) if threshold < 65536 else 0.0, dtype=wide.dtype)
    return torch.where(keep, wide * scale, torch.zeros((), dtype=wide.dtype)).to(x.dtype)


# --------------------------------------------------------------------------- e4m3 with a scale for each block of 128
def e4m3(v):
    """The nearest e4m3 value of each |v| <= 448, to even between two: steps of 2^-3 of the power of two below v, of 2^-9
    under 2^-6."""
    exponent = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6)))
    step = 2.0 ** (exponent - 3)
    return np.round(v / step) * step


def quantize_fp8(x):
    """(rows, k) in 64 bits -> (values of q, exponents e of the blocks' scales)."""
    rows, k = x.shape
    blocks = -(-k // 128)
    b = np.zeros((rows, blocks * 128))
    b[:, :k] = x
    b = b.reshape(rows, blocks, 128)
    amax = np.abs(b).max(axis=2)
    m, e = np.frexp(amax)                       # 448 = 0.875 * 2^9
    e = np.clip(np.where(m <= 0.875, e - 9, e - 8), -127, 127)
    e = np.where(amax == 0, -127, e)
    return e4m3(b / 2.0 ** e[:, :, None]).reshape(rows, blocks * 128), e


def dequantize_fp8(q, e):
    return (q.reshape(q.shape[0], -1, 128) * 2.0 ** e[:, :, None].astype(np.float64)).reshape(q.shape)


def matmul_fp8(x, wq, we, bias, relu, dtype):
    """The product of the quantised operands, and how far a kernel may be from it.  Each block's product and each sum of
    blocks is rounded by at most a step of 32 bits (2^-23) of the sum of magnitudes, bias and result once.  For 16-bit
    results the matrix instruction also cuts the products of each eight elements off 13 bits below the largest of them:
    up to seven times 2^-13 of it, 16 eights a block, none larger than the block's largest product."""
    xd, wd = dequantize_fp8(*quantize_fp8(x)), dequantize_fp8(wq, we)
    y = xd @ wd.T
    bound = (we.shape[1] + 2) * 2.0 ** -23 * (np.abs(xd) @ np.abs(wd).T)
    if dtype != torch.float32:
        for b in range(0, xd.shape[1], 128):
            most = np.abs(xd[:, b:b + 128]).max(axis=1)[:, None] * np.abs(wd[:, b:b + 128]).max(axis=1)[None]
            bound += 16 * 7 * 2.0 ** -13 * most
    if bias is not None:
        y = y + bias
        bound = bound + 2.0 ** -24 * np.abs(y)
    y = np.where(y > 0, y, 0) if relu else y
    return y, bound + HALF_STEP[dtype] * np.abs(y) + TINY[dtype]
