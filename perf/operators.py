"""Cases of the operators that train and serve a network's normalisation, dropout and FC head, with their plain forms.

  gn        group norm with an activation: forward (y, mean, 1/std) and backward (dgamma, dbeta, dx)
  dropout   dropout whose mask is a function of (seed, offset, index) and is never stored; the backward pass is the same map of dy
  fp8       FC product in e4m3: activations scaled by blocks of 128 on the way, weights laid out once

``run`` computes a case in elementary torch operations, or, where ``own`` is true, through ``pydtnn_amd.ops``.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f64": 8, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # the smallest block of a test network: latency of one call
        {"name": "gn fwd 2x8x8x16", "op": "gn", "pass": "forward", "dtype": "f32", "n": 2, "h": 8, "w": 8, "c": 16,
         "groups": 4, "act": "relu"},
        # the output of AlexNet's first convolution: odd planes, 12 channels to a group
        {"name": "gn fwd 64x55x55x96", "op": "gn", "pass": "forward", "dtype": "bf16", "n": 64, "h": 55, "w": 55,
         "c": 96, "groups": 8, "act": "silu"},
        # the activations of a 3x3 256 -> 256 layer at batch 64, the largest tensors that the framework's benchmark has
        {"name": "gn fwd 64x56x56x256", "op": "gn", "pass": "forward", "dtype": "f32", "n": 64, "h": 56, "w": 56,
         "c": 256, "groups": 32, "act": "relu"},
        # training in double precision
        {"name": "gn bwd 16x28x28x128", "op": "gn", "pass": "backward", "dtype": "f64", "n": 16, "h": 28, "w": 28,
         "c": 128, "groups": 32, "act": "silu"},
        {"name": "gn bwd 64x56x56x256", "op": "gn", "pass": "backward", "dtype": "f32", "n": 64, "h": 56, "w": 56,
         "c": 256, "groups": 32, "act": "relu"},
        # VGG16's head in training
        {"name": "dropout fwd 64x4096", "op": "dropout", "pass": "forward", "dtype": "f32", "n": 64 * 4096, "rate": 0.5},
        # an odd number of elements in 16 bits
        {"name": "dropout bwd 33x25087", "op": "dropout", "pass": "backward", "dtype": "bf16", "n": 33 * 25087,
         "rate": 0.1},
        {"name": "dropout fwd 64x56x56x256", "op": "dropout", "pass": "forward", "dtype": "f32",
         "n": 64 * 56 * 56 * 256, "rate": 0.2},
        # VGG16's three FC layers: one image through the last, a batch of 16 through the first
        {"name": "fp8 1x4096x1000", "op": "fp8", "dtype": "f32", "m": 1, "k": 4096, "n": 1000, "relu": False},
        {"name": "fp8 16x25088x4096", "op": "fp8", "dtype": "f32", "m": 16, "k": 25088, "n": 4096, "relu": True},
        # ragged in every extent
        {"name": "fp8 777x2049x1003", "op": "fp8", "dtype": "f16", "m": 777, "k": 2049, "n": 1003, "relu": True},
        # a large batch: bound by the matrix cores
        {"name": "fp8 4096x4096x4096", "op": "fp8", "dtype": "bf16", "m": 4096, "k": 4096, "n": 4096, "relu": False},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["gn", "gn", "dropout", "fp8", "fp8"])
    most = 64 * 56 * 56 * 256 * 4        # bytes of the largest listed tensor
    if op == "gn":
        dtype = rng.choice(["f32", "f32", "bf16", "f16", "f64"])
        groups, cg = _spread(rng, 1, 64), _spread(rng, 1, 64)
        while groups * cg > 1024:
            cg = max(1, cg // 2)
        n, h, w = _spread(rng, 1, 64), _spread(rng, 1, 112), _spread(rng, 1, 112)
        if h * w * cg < 16:      # the gradient of a group of two or three elements is nothing but rounding
            h = w = 4
        while n * h * w * groups * cg * ITEM[dtype] > most:
            n, h = max(1, n // 2), max(1, (h + 1) // 2)
        return {"op": "gn", "pass": rng.choice(["forward", "backward"]), "dtype": dtype, "n": n, "h": h, "w": w,
                "c": groups * cg, "groups": groups, "act": rng.choice(["", "relu", "silu"])}
    if op == "dropout":
        dtype = rng.choice(["f32", "f32", "bf16", "f16", "f64"])
        return {"op": "dropout", "pass": rng.choice(["forward", "backward"]), "dtype": dtype,
                "n": _spread(rng, 1000, most // ITEM[dtype]), "rate": rng.choice([0.05, 0.1, 0.2, 0.25, 0.5, 0.75])}
    m, k, n = _spread(rng, 1, 4096), _spread(rng, 16, 25088), _spread(rng, 10, 4096)
    while m * k * n > 4096 ** 3:
        m //= 2
    return {"op": "fp8", "dtype": rng.choice(["f32", "bf16", "f16"]), "m": m, "k": k, "n": n,
            "relu": rng.random() < 0.5}


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "gn":
        # activations of a convolution: a mean and a spread of their own in each channel
        shape, c = (case["n"], case["h"], case["w"], case["c"]), case["c"]
        vector = torch.float64 if dtype == torch.float64 else torch.float32
        scale = torch.rand(c, generator=g, device="cuda") + 0.5
        shift = torch.randn(c, generator=g, device="cuda")
        s["x"] = (_normal(g, shape, torch.float32) * scale + shift).to(dtype)
        s["gamma"] = (torch.rand(c, generator=g, device="cuda") + 0.5).to(vector)
        s["beta"] = (torch.randn(c, generator=g, device="cuda") * 0.3).to(vector)
        if case["pass"] == "backward":
            s["dy"] = _normal(g, shape, dtype)
            mean, inv_std = _gn_statistics(_groups(s["x"].double(), case["groups"]))
            s["mean"], s["inv_std"] = mean.to(vector), inv_std.to(vector)
    elif case["op"] == "dropout":
        s["x"] = _normal(g, (case["n"],), dtype)
        s["seed"], s["offset"] = seed * 2654435761 % (1 << 63), seed % 1000 + (seed << 20)
    else:
        s["x"] = _normal(g, (case["m"], case["k"]), dtype).relu_()    # what the layer before it hands over
        w = torch.randn((case["n"], case["k"]), generator=g, device="cuda") * math.sqrt(2.0 / case["k"])
        s["wq"], s["ws"] = _quantize(w)
        s["bias"] = torch.randn(case["n"], generator=g, device="cuda") * 0.1
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _groups(x, groups):
    """(n, h, w, c) as (n, pixels, groups, channels of a group)."""
    return x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def _gn_statistics(x):
    mean = x.mean(dim=(1, 3))
    var = (x - mean[:, None, :, None]).square().mean(dim=(1, 3))
    return mean, 1.0 / torch.sqrt(var + EPS)


def _gn_forward(s):
    case, x = s["case"], s["x"]
    xg = _groups(x.to(s["gamma"].dtype), case["groups"])
    mean, inv_std = _gn_statistics(xg)
    gamma, beta = s["gamma"].view(case["groups"], -1), s["beta"].view(case["groups"], -1)
    z = (xg - mean[:, None, :, None]) * inv_std[:, None, :, None] * gamma + beta
    if case["act"] == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif case["act"] == "silu":
        z = z / (1 + torch.exp(-z))
    return {"y": z.reshape(x.shape).to(x.dtype), "mean": mean, "inv_std": inv_std}


def _gn_backward(s):
    case, x, groups = s["case"], s["x"], s["case"]["groups"]
    mean, inv_std = s["mean"][:, None, :, None], s["inv_std"][:, None, :, None]
    gamma, beta = s["gamma"].view(groups, -1), s["beta"].view(groups, -1)
    xg, dz = _groups(x.to(mean.dtype), groups), _groups(s["dy"].to(mean.dtype), groups)
    xn = (xg - mean) * inv_std
    if case["act"] == "relu":     # the border of the rectifier, in 64 bits: one element on its wrong side is a whole dy off
        z = (xg.double() - mean.double()) * inv_std.double() * gamma.double() + beta.double()
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    elif case["act"] == "silu":
        z = xn * gamma + beta
        p = 1 / (1 + torch.exp(-z))
        dz = dz * (p * (1 + z * (1 - p)))
    dgamma, dbeta = (dz * xn).sum(dim=(0, 1)).reshape(-1), dz.sum(dim=(0, 1)).reshape(-1)
    dxn = dz * gamma
    a, b = dxn.mean(dim=(1, 3), keepdim=True), (dxn * xn).mean(dim=(1, 3), keepdim=True)
    dx = (dxn - a - xn * b) * inv_std
    return {"dgamma": dgamma, "dbeta": dbeta, "dx": dx.reshape(x.shape).to(x.dtype)}


def _philox(calls, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): the key is the
    seed, the counter the number of the call and the offset; int64 tensors hold the 32-bit words."""
    low = 0xFFFFFFFF
    c0, c1 = calls & low, calls >> 32
    c2, c3 = torch.full_like(calls, offset & low), torch.full_like(calls, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57        # 64 bits each; the sign is shifted in and masked away
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), dim=1)


def _dropout(s):
    x, threshold = s["x"], round(s["case"]["rate"] * 65536)
    words = _philox(torch.arange((x.numel() + 7) // 8, device=x.device), s["seed"], s["offset"])
    u = torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:x.numel()].reshape(x.shape)
    wide = x if x.dtype == torch.float64 else x.float()
    return torch.where(u >= threshold, wide * (65536 / (65536 - threshold)), torch.zeros_like(wide)).to(x.dtype)


def _quantize(x):
    """(rows, k) -> e4m3 values (rows, k to a multiple of 128) and the biased exponents of the blocks' scales (rows, blocks
    to a multiple of 4).  A scale is the smallest power of two that brings its block within the largest e4m3 value, 448."""
    rows, k = x.shape
    blocks = (k + 127) // 128
    b = torch.nn.functional.pad(x.float(), (0, blocks * 128 - k)).view(rows, blocks, 128)
    amax = b.abs().amax(dim=2)
    m, e = torch.frexp(amax)                   # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-127, 127)
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    q = torch.ldexp(b, -e[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks * 128)
    scales = torch.full((rows, (blocks + 3) // 4 * 4), 127, dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return q, scales


def _dequantize(q, scales):
    blocks = q.shape[1] // 128
    scale = torch.ldexp(torch.ones((), device=q.device), scales[:, :blocks].int() - 127)
    return (q.float().view(-1, blocks, 128) * scale[:, :, None]).view(q.shape)


def _fp8(s):
    y = _dequantize(*_quantize(s["x"])) @ _dequantize(s["wq"], s["ws"]).t() + s["bias"]
    if s["case"]["relu"]:
        y = torch.where(y > 0, y, torch.zeros_like(y))
    return y.to(s["x"].dtype)


def run(s):
    case = s["case"]
    if own:
        from pydtnn_amd import ops
        if case["op"] == "gn" and case["pass"] == "forward":
            y, mean, inv_std = ops.gn_forward(s["x"], s["gamma"], s["beta"], case["groups"], EPS, case["act"])
            return {"y": y, "mean": mean, "inv_std": inv_std}
        if case["op"] == "gn":
            dgamma, dbeta, dx = ops.gn_backward(s["dy"], s["x"], s["gamma"], s["beta"], s["mean"], s["inv_std"],
                                                case["groups"], case["act"])
            return {"dgamma": dgamma, "dbeta": dbeta, "dx": dx}
        if case["op"] == "dropout":
            f = ops.dropout if case["pass"] == "forward" else ops.dropout_backward
            return f(s["x"], case["rate"], s["seed"], s["offset"])
        return ops.matmul_fp8(s["x"], s["wq"], s["ws"], bias=s["bias"], relu=case["relu"])
    if case["op"] == "gn":
        return _gn_forward(s) if case["pass"] == "forward" else _gn_backward(s)
    return _dropout(s) if case["op"] == "dropout" else _fp8(s)


def work(case):
    item = ITEM[case["dtype"]]
    if case["op"] == "gn":
        numel = case["n"] * case["h"] * case["w"] * case["c"]
        small = 2 * case["n"] * case["groups"] + 2 * case["c"]
        if case["pass"] == "forward":
            return {"bytes": 2 * numel * item + small * max(4, item), "flops": 8 * numel}
        return {"bytes": 3 * numel * item + (small + 2 * case["c"]) * max(4, item), "flops": 14 * numel}
    if case["op"] == "dropout":
        return {"bytes": 2 * case["n"] * item, "flops": case["n"]}
    m, k, n = case["m"], case["k"], case["n"]
    return {"bytes": m * k * item + n * k + n * ((k + 127) // 128) + 4 * n + m * n * item, "flops": 2 * m * k * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_gn(s):
    """From sums of each channel, channel by channel joined to groups."""
    case = s["case"]
    n, c, g = case["n"], case["c"], case["groups"]
    x = s["x"].double().reshape(n, -1, c)
    gamma, beta = s["gamma"].double(), s["beta"].double()

    def each(t):      # (n, groups) -> (n, 1, c)
        return t.repeat_interleave(c // g, dim=1)[:, None, :]

    def joined(t):    # (n, c) -> mean over each group's channels and pixels
        return t.view(n, g, c // g).sum(dim=2) / (x.shape[1] * (c // g))

    if case["pass"] == "forward":
        mean = joined(x.sum(dim=1))
        d = x - each(mean)
        inv_std = (joined((d * d).sum(dim=1)) + EPS).rsqrt()
        z = torch.addcmul(beta, d * each(inv_std), gamma)
        if case["act"] == "relu":
            z = z.clamp_min(0)
        elif case["act"] == "silu":
            z = z * torch.sigmoid(z)
        return {"y": z.reshape(s["x"].shape), "mean": mean, "inv_std": inv_std}
    r = each(s["inv_std"].double())
    xn = (x - each(s["mean"].double())) * r
    dz = s["dy"].double().reshape(n, -1, c)
    if case["act"]:
        z = xn * gamma + beta
        if case["act"] == "relu":
            dz = dz * (z > 0)
        else:
            p = torch.sigmoid(z)
            dz = dz * (p + z * p * (1 - p))
    s1, s2 = dz.sum(dim=1), (dz * xn).sum(dim=1)
    dx = r * (gamma * dz - each(joined(s1 * gamma)) - xn * each(joined(s2 * gamma)))
    return {"dgamma": s2.sum(dim=0), "dbeta": s1.sum(dim=0), "dx": dx.reshape(s["x"].shape)}


def _exact_dropout(s):
    n, seed, offset = s["case"]["n"], s["seed"], s["offset"]
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    call = np.arange((n + 7) // 8, dtype=np.uint64)
    ctr = [call & low, call >> half, np.full_like(call, offset & 0xFFFFFFFF), np.full_like(call, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> half) ^ ctr[1] ^ np.uint64(key[0]), b & low, (a >> half) ^ ctr[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    u = np.stack(ctr, axis=1).astype(np.uint32).view(np.uint16).reshape(-1)[:n]      # little endian: low halves first
    dropped = math.floor(s["case"]["rate"] * 65536 + 0.5)
    x = s["x"].double()
    keep = torch.from_numpy((u >= dropped).astype(np.float64)).to(x.device)
    return x * keep / (1 - dropped / 65536)


def _exact_e4m3(v):
    """The values that e4m3 holds for v, |v| <= 448: steps of 2^-3 of the power of two below v, 2^-9 under 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_fp8(s):
    x = s["x"].double()
    m, k = x.shape
    kp = (k + 127) // 128 * 128
    x = torch.cat((x, x.new_zeros(m, kp - k)), dim=1).view(m, kp // 128, 128)
    top = x.abs().amax(dim=2, keepdim=True) / 448
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0 ** -127))))
    x = (_exact_e4m3(x / scale) * scale).view(m, kp)
    w = s["wq"].double().view(-1, kp // 128, 128) * torch.exp2(s["ws"][:, :kp // 128].double() - 127)[:, :, None]
    y = x @ w.view(-1, kp).t() + s["bias"].double()
    return y.clamp_min(0) if s["case"]["relu"] else y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gn":
        return _exact_gn(s)
    return _exact_dropout(s) if case["op"] == "dropout" else _exact_fp8(s)
