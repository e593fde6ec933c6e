"""GPU tests of the operators for several element types against their plain 64-bit forms (operator_oracles.py)."""
import numpy as np
import pytest
import torch

import operator_oracles as oo
from gpu_util import announce

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def pd():
    import pydtnn_amd
    from pydtnn_amd import native
    native.lib()
    return pydtnn_amd


@pytest.fixture(scope="module")
def ops(pd):
    from pydtnn_amd import ops
    return ops


def wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def within(got, ref, bound, what):
    got = oo.host64(got)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    over = np.abs(got - ref) - bound
    assert np.all(np.isfinite(got)), f"{what}: not finite"
    assert np.all(over <= 0), f"{what}: {np.max(np.abs(got - ref)):.3e} off, {np.max(over):.3e} over its bound"


def misaligned(t):
    """The same values one element behind a 16-byte boundary."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    buf[1:].copy_(t.reshape(-1))
    return buf[1:].view(t.shape)


# --------------------------------------------------------------------------- group normalisation
# (batch, spatial extents, channels, groups)
GN_SHAPES = [
    (1, (1, 1), 1, 1),             # a group of one element
    (3, (), 8, 2),                 # a matrix
    (2, (7, 7), 64, 32),           # two channels to a group
    (2, (5, 3), 30, 5),            # channels that no pack of four divides
    (3, (9, 11), 96, 8),           # groups of 12: packs of 8 straddle them
    (5, (33,), 16, 16),            # a group to each channel
    (1, (3, 3), 2048, 4),          # more packs than threads: slabs of whole groups
    (1, (2, 2), 1030, 2),          # groups wider than a workgroup, no packs
    (2, (2, 1), 4100, 1),          # one group over a long row
    (2, (65, 63), 8, 2),           # many pixels: runs
    (1, (40, 41), 320, 32),        # runs of an image with idle threads
    (1500, (2, 2), 4, 2),          # many small images
    (2, (28, 28), 64, 8),          # slabs that a workgroup's registers hold: of several sizes of workgroup
    (1, (27, 29), 48, 1),
    (3, (14, 13), 160, 10),
    (1, (56, 55), 32, 4),
    (1, (56, 57), 96, 6),
    (2, (90, 80), 32, 16),         # and slabs that they do not
]


def gn_inputs(shape, dtype, nhwc, seed, offset=1.0):
    n, spatial, c, groups = shape
    g = torch.Generator().manual_seed(seed)
    full = (n, *spatial, c) if nhwc else (n, c, *spatial)
    x = (torch.randn(full, generator=g) * 1.5 + offset).to(dtype).cuda()
    dy = torch.randn(full, generator=g).to(dtype).cuda()
    gamma = (torch.randn(c, generator=g)).to(wide(dtype)).cuda()
    beta = (torch.randn(c, generator=g) * 0.5).to(wide(dtype)).cuda()
    if c > 3:
        gamma[1] = 0          # a channel that is its shift alone
        beta[2] = 0
    return x, dy, gamma, beta, groups


def check_gn(ops, x, dy, gamma, beta, groups, activation, nhwc, eps=1e-5):
    dtype = x.dtype
    hx, hdy, hg, hb = (oo.host64(t) for t in (x, dy, gamma, beta))
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, eps, activation, nhwc)
    ref = oo.gn_forward(hx, hg, hb, groups, eps, activation, nhwc)
    bounds = oo.gn_forward_bounds(hx, hg, hb, groups, eps, nhwc, ref[0], dtype)
    assert y.dtype == dtype and mean.dtype == inv_std.dtype == wide(dtype)
    for got, r, b, what in zip((y, mean, inv_std), ref, bounds, ("y", "mean", "inv_std")):
        within(got, r, b, what)
    hm, hi = oo.host64(mean), oo.host64(inv_std)
    dgamma, dbeta, dx = ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, activation, nhwc)
    ref = oo.gn_backward(hdy, hx, hg, hb, hm, hi, groups, activation, nhwc)
    bounds = oo.gn_backward_bounds(hdy, hx, hg, hb, hm, hi, groups, activation, nhwc, ref[2], dtype)
    for got, r, b, what in zip((dgamma, dbeta, dx), ref, bounds, ("dgamma", "dbeta", "dx")):
        within(got, r, b, what)
    again = ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, activation, nhwc, need_dx=False)
    assert again[2] is None and torch.equal(again[0], dgamma) and torch.equal(again[1], dbeta)


@pytest.mark.parametrize("nhwc", [True, False], ids=["last", "first"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", GN_SHAPES, ids=str)
def test_group_norm(ops, shape, dtype, nhwc):
    for activation in ("", "relu", "silu"):
        announce("group norm", shape, dtype, nhwc, activation)
        check_gn(ops, *gn_inputs(shape, dtype, nhwc, 5), activation, nhwc)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, (225, 223), 6, 2), (2, (47, 43), 5, 1), (3, (13, 11), 7, 7), (2, (3, 1), 6, 3)], ids=str)
def test_group_norm_of_planes_of_odd_extents(ops, shape, dtype):
    """Planes and groups that no pack divides and that start off the boundaries of packs, of sizes for a workgroup, a wave and
    a part of one; forward in two passes."""
    announce("group norm, odd planes", shape, dtype)
    x, dy, gamma, beta, groups = gn_inputs(shape, dtype, False, 7)
    check_gn(ops, x, dy, gamma, beta, groups, "relu", False)
    check_gn(ops, misaligned(x), misaligned(dy), gamma, beta, groups, "silu", False)


@pytest.mark.parametrize("nhwc", [True, False], ids=["last", "first"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(64, (13, 17), 128, 8), (64, (23, 23), 128, 4), (30, (18, 17), 544, 17)], ids=str)
def test_group_norm_of_many_slabs_of_whole_lines(ops, shape, dtype, nhwc):
    """Images enough for a slab of whole lines to each compute unit, of sizes that take the larger workgroups."""
    announce("group norm, many slabs", shape, dtype, nhwc)
    check_gn(ops, *gn_inputs(shape, dtype, nhwc, 6), "silu" if shape[0] == 30 else "relu", nhwc)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_group_norm_of_values_far_from_zero(ops, dtype, offset):
    announce("group norm far from zero", dtype, offset)
    x, dy, gamma, beta, groups = gn_inputs((2, (13, 9), 24, 3), dtype, True, 6, offset)
    check_gn(ops, x, dy, gamma, beta, groups, "silu", True)
    x, dy, gamma, beta, groups = gn_inputs((2, (13, 9), 24, 3), dtype, False, 6, offset)
    check_gn(ops, x, dy, gamma, beta, groups, "relu", False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_group_norm_of_a_constant_group(ops, dtype):
    """No spread at all: y is the shift, and the gradient stays finite."""
    announce("group norm constant", dtype)
    x, dy, gamma, beta, groups = gn_inputs((2, (4, 5), 16, 4), dtype, True, 7)
    x[0] = 2.5
    check_gn(ops, x, dy, gamma, beta, groups, "", True, eps=1e-3)
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, 1e-3)
    assert torch.equal(y[0], beta.to(dtype).expand_as(y[0])) and torch.all(mean[0] == 2.5)


def test_group_norm_of_one_element_has_no_gradient(ops):
    announce("group norm of single elements")
    x, dy, gamma, beta, groups = gn_inputs((4, (), 6, 6), torch.float32, True, 8)
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups)
    assert torch.equal(y, beta.expand_as(y))
    assert torch.count_nonzero(ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups)[2]) == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("nhwc", [True, False], ids=["last", "first"])
def test_group_norm_of_tensors_off_their_alignment(ops, dtype, nhwc):
    announce("group norm misaligned", dtype, nhwc)
    x, dy, gamma, beta, groups = gn_inputs((2, (6, 7), 64, 8), dtype, nhwc, 9)
    check_gn(ops, misaligned(x), misaligned(dy), misaligned(gamma), misaligned(beta), groups, "relu", nhwc)
    check_gn(ops, x, misaligned(dy), gamma, beta, groups, "silu", nhwc)


def test_group_norm_of_strided_views(ops):
    announce("group norm strided")
    x, dy, gamma, beta, groups = gn_inputs((4, (6, 10), 32, 8), torch.float32, True, 10)
    for view in (lambda t: t[::2], lambda t: t[:, :, ::2], lambda t: t.transpose(1, 2), lambda t: t[..., :16]):
        c = view(x).shape[-1]
        check_gn(ops, view(x), view(dy), gamma[:c], beta[:c], groups, "relu", True)


def test_group_norm_of_nothing(ops):
    announce("group norm of no images")
    x, dy, gamma, beta, groups = gn_inputs((0, (6, 10), 32, 8), torch.float32, True, 11)
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups)
    assert y.shape == x.shape and mean.shape == (0, 8)
    dgamma, dbeta, dx = ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups)
    assert torch.count_nonzero(dgamma) == torch.count_nonzero(dbeta) == 0 and dx.shape == x.shape


def test_group_norm_keeps_what_is_not_a_number_in_its_group(ops):
    announce("group norm of NaN")
    x, dy, gamma, beta, groups = gn_inputs((2, (6, 6), 16, 4), torch.float32, True, 12)
    clean = ops.gn_forward(x, gamma, beta, groups)[0]
    x[0, 2, 3, 5] = float("nan")
    x[1, 2, 3, 5] = float("inf")
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups)
    assert torch.isnan(y[..., 4:8]).all() and not torch.isnan(mean[:, [0, 2, 3]]).any()
    rest = [c for c in range(16) if not 4 <= c < 8]
    assert torch.equal(y[..., rest], clean[..., rest])


@pytest.mark.parametrize("activation", ["", "silu"])
def test_group_norm_gradients_are_the_slopes_of_the_forward_kernel(ops, activation):
    """Central differences of the kernel itself in float64: h^2 times the third derivative and 1e-16 |loss| / h."""
    announce("group norm differences", activation)
    x, dy, gamma, beta, groups = gn_inputs((2, (5, 6), 12, 3), torch.float64, True, 13)

    def loss(x, gamma, beta):
        return float((ops.gn_forward(x, gamma, beta, groups, 1e-5, activation)[0] * dy).sum())

    _, mean, inv_std = ops.gn_forward(x, gamma, beta, groups)
    grads = ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, activation)
    h = 1e-5
    for which, grad in ((1, grads[0]), (2, grads[1]), (0, grads[2])):
        args = [x, gamma, beta]
        v = torch.randn(args[which].shape, generator=torch.Generator().manual_seed(which), dtype=torch.float64).cuda()
        up, down = list(args), list(args)
        up[which], down[which] = args[which] + h * v, args[which] - h * v
        assert abs((loss(*up) - loss(*down)) / (2 * h) - float((grad * v).sum())) < 1e-6


def test_group_norm_of_a_tensor_of_more_than_2_to_31_elements(ops):
    announce("group norm beyond 32 bits")
    images, pixels, c, groups = 9, 1 << 18, 1024, 32
    x = torch.empty((images, pixels, c), dtype=torch.bfloat16, device="cuda")
    for i in range(images):
        x[i].normal_(generator=torch.Generator(device="cuda").manual_seed(i))
    gamma = torch.rand(c, device="cuda") + 0.5
    beta = torch.randn(c, device="cuda")
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, activation="relu")
    alone = ops.gn_forward(x[-1:].clone(), gamma, beta, groups, activation="relu")
    # the same image by itself: its runs are others, so its sums are rounded in another order
    assert torch.allclose(mean[-1:], alone[1], rtol=0, atol=1e-6)
    assert torch.allclose(inv_std[-1:], alone[2], rtol=1e-5, atol=0)
    assert torch.allclose(y[-1].float(), alone[0][0].float(), rtol=2 ** -7, atol=1e-4)
    dx = ops.gn_backward(y, x, gamma, beta, mean, inv_std, groups, "relu")[2]
    dx1 = ops.gn_backward(y[-1:].clone(), x[-1:].clone(), gamma, beta, mean[-1:].clone(), inv_std[-1:].clone(), groups,
                          "relu")[2]
    assert torch.allclose(dx[-1].float(), dx1[0].float(), rtol=2 ** -7, atol=1e-4)


# --------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("count", [1, 7, 8, 9, 2047, 2049, 100003])
def test_dropout_is_its_plain_form_bit_for_bit(ops, dtype, count):
    g = torch.Generator().manual_seed(count)
    x = torch.randn(count, generator=g, dtype=torch.float64).to(dtype).cuda()
    for rate, seed, offset in ((0.5, 0, 0), (0.1, 12345, 7), (0.3, (1 << 64) - 3, (1 << 40) + 5), (1 / 131072, 1, 2),
                               (3 / 131072, 1, 2), (0.0, 3, 4), (1.0, 3, 4), (0.999, 5, 6)):
        announce("dropout", dtype, count, rate, seed, offset)
        ref = oo.dropout(x, rate, seed, offset)
        assert torch.equal(ops.dropout(x, rate, seed, offset).cpu(), ref)
        assert torch.equal(ops.dropout(misaligned(x), rate, seed, offset).cpu(), ref)
        assert torch.equal(ops.dropout_backward(x, rate, seed, offset).cpu(), ref)
        there = torch.tensor([offset if offset < 1 << 63 else offset - (1 << 64)], device="cuda")
        assert torch.equal(ops.dropout(x, rate, seed, there).cpu(), ref)


def test_dropout_drops_what_is_not_a_number(ops):
    announce("dropout of NaN")
    x = torch.full((4096,), float("nan"), device="cuda")
    x[1::2] = float("inf")
    keep = torch.from_numpy(oo.dropout_numbers(0, 4096, 9, 1) >= 32768).cuda()
    y = ops.dropout(x, 0.5, 9, 1)
    assert torch.all(y[~keep] == 0) and torch.isnan(y[::2][keep[::2]]).all() and torch.isinf(y[1::2][keep[1::2]]).all()


def test_dropout_of_shapes_and_strides(ops):
    announce("dropout shapes")
    x = torch.randn(6, 10, 14, device="cuda")
    flat = ops.dropout(x.reshape(-1), 0.4, 2, 3)
    assert torch.equal(ops.dropout(x, 0.4, 2, 3).reshape(-1), flat)
    t = x.transpose(0, 2)
    assert torch.equal(ops.dropout(t, 0.4, 2, 3), ops.dropout(t.contiguous(), 0.4, 2, 3))
    assert ops.dropout(x[:0], 0.4, 2, 3).shape == (0, 10, 14)


@pytest.mark.parametrize("rate", [0.05, 0.5, 0.9])
def test_dropout_keeps_the_mean(ops, rate):
    """2^22 draws: the share kept is within 5 standard deviations of its probability."""
    announce("dropout share", rate)
    n = 1 << 22
    y = ops.dropout(torch.ones(n, device="cuda"), rate, 77, 1)
    threshold = round(rate * 65536)
    p = 1 - threshold / 65536
    kept = float((y != 0).double().mean())
    assert abs(kept - p) < 5 * (p * (1 - p) / n) ** 0.5
    other = ops.dropout(torch.ones(n, device="cuda"), rate, 77, 2)
    both = float(((y != 0) & (other != 0)).double().mean())
    assert abs(both - p * p) < 5 * (p * p * (1 - p * p) / n) ** 0.5


def test_dropout_of_more_than_2_to_31_elements(ops):
    announce("dropout beyond 32 bits")
    n = (1 << 31) + 8 * 1000 + 3
    y = ops.dropout(torch.ones(n, dtype=torch.bfloat16, device="cuda"), 0.5, 4, 5)
    first = (1 << 31) - 8 * 1000
    u = oo.dropout_numbers(first, n - first, 4, 5)
    assert np.array_equal(oo.host64(y[first:]), np.where(u >= 32768, 2.0, 0.0))


def test_dropout_draws_anew_at_each_replay_of_a_captured_graph(ops):
    announce("dropout in a graph")
    x = torch.randn(5000, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.dropout(x, 0.5, 11, step)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step += 1
        y = ops.dropout(x, 0.5, 11, step)
        dx = ops.dropout_backward(y, 0.5, 11, step)
    for i in range(1, 6):
        graph.replay()
        torch.cuda.synchronize()
        ref = oo.dropout(x, 0.5, 11, i)
        assert torch.equal(y.cpu(), ref) and torch.equal(dx.cpu(), oo.dropout(y, 0.5, 11, i))
        ops.dropout(x, 0.3, 1, i)          # the program's own work between replays


def test_group_norm_in_graphs_of_their_own(ops):
    """Two captured graphs and eager calls of other sizes between their replays."""
    announce("group norm in graphs")
    cases = [gn_inputs((3, (30, 31), 64, 8), torch.float32, True, 21), gn_inputs((2, (9, 8), 32, 4), torch.float32, True, 22)]
    eager, graphs = [], []
    for x, dy, gamma, beta, groups in cases:
        y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, activation="relu")
        eager.append((y, *ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, "relu")))
    torch.cuda.synchronize()
    for x, dy, gamma, beta, groups in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, activation="relu")
            out = (y, *ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, "relu"))
        graphs.append((graph, out))
    big = gn_inputs((4, (64, 64), 128, 8), torch.float32, True, 23)
    for _ in range(4):
        for (graph, out), ref in zip(graphs, eager):
            for t in out:
                t.zero_()
            graph.replay()
            ops.gn_forward(big[0], big[2], big[3], big[4])
            torch.cuda.synchronize()
            for t, r in zip(out, ref):
                assert torch.equal(t, r)


def test_calls_on_two_streams_at_once(ops):
    announce("two streams")
    a = gn_inputs((4, (56, 57), 64, 8), torch.float32, True, 24)
    b = gn_inputs((3, (41, 40), 96, 8), torch.float32, True, 25)
    refs = []
    for x, dy, gamma, beta, groups in (a, b):
        y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, activation="silu")
        refs.append((y, *ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, "silu"), ops.dropout(x, 0.5, 1, 2)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        outs = []
        for stream, (x, dy, gamma, beta, groups) in zip(streams, (a, b)):
            with torch.cuda.stream(stream):
                y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, activation="silu")
                outs.append((y, *ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, "silu"),
                             ops.dropout(x, 0.5, 1, 2)))
        torch.cuda.synchronize()
        for out, ref in zip(outs, refs):
            assert all(torch.equal(t, r) for t, r in zip(out, ref))


# --------------------------------------------------------------------------- e4m3 with a scale for each block of 128
FP8_DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def fp8_matrix(rows, k, dtype, seed, spread=True):
    """Values whose size changes from block to block and from row to row, a block of zeros, values at the edges."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    if spread:
        x *= torch.exp2(torch.randint(-6, 5, (rows, -(-k // 128)), generator=g).float()).repeat_interleave(128, 1)[:, :k]
        x[0, :128] = 0
        x[-1, 0] = 448.0                       # the largest e4m3 value: its block keeps scale 1 or above
        x[-1, k // 2] = 2.0 ** -9
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", FP8_DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (2, 128), (5, 129), (1, 511), (7, 512), (4, 513), (9, 2049), (33, 1000)],
                         ids=str)
def test_quantization_is_its_plain_form_bit_for_bit(ops, shape, dtype):
    announce("quantize", shape, dtype)
    x = fp8_matrix(*shape, dtype, sum(shape))
    ref, e = oo.quantize_fp8(oo.host64(x))
    for t in (x, misaligned(x), x.t().contiguous().t()):
        q, scales = ops.quantize_fp8(t)
        assert np.array_equal(oo.host64(q), ref)
        got = scales.cpu().numpy().astype(np.int64) - 127
        assert np.array_equal(got[:, :e.shape[1]], e) and np.all(got[:, e.shape[1]:] == 0)


def test_quantization_of_the_smallest_and_largest_values(ops):
    """Scales at both ends of their range, values that a scale's edge decides, and ties."""
    announce("quantize edges")
    f = torch.finfo(torch.float32)
    rows = [448.0, 448.0 * (1 + 2 ** -23), 447.99997, 224.0, f.max, f.tiny, 2.0 ** -149, 448 * 2.0 ** -127, 1.0, 17.0, 19.0,
            2.0 ** -10, 3 * 2.0 ** -10]
    x = torch.zeros(len(rows), 256)
    x[:, 0] = torch.tensor(rows, dtype=torch.float64).float()
    x[:, 5] = -x[:, 0] / 16 * 1.0625
    x[:, 130] = x[:, 0] * 0.3
    q, scales = ops.quantize_fp8(x.cuda())
    ref, e = oo.quantize_fp8(oo.host64(x))
    assert np.array_equal(scales.cpu().numpy()[:, :2].astype(np.int64) - 127, e)
    assert np.array_equal(oo.host64(q), ref)


# (m, n, k): from one element to ragged extents, few rows, many rows, long k
FP8_SHAPES = [(1, 1, 1), (1, 1000, 4096), (2, 10, 130), (3, 63, 128), (7, 257, 513), (16, 64, 2048), (17, 16, 127),
              (16, 96, 25088), (31, 100, 384), (33, 130, 1000), (64, 256, 1024), (65, 31, 640), (100, 1003, 777),
              (129, 257, 2049), (257, 511, 300), (300, 640, 512), (512, 512, 4096), (1025, 384, 256)]


@pytest.mark.parametrize("dtype", FP8_DTYPES, ids=str)
@pytest.mark.parametrize("shape", FP8_SHAPES, ids=str)
def test_matmul_fp8(ops, shape, dtype):
    m, n, k = shape
    announce("matmul_fp8", shape, dtype)
    # weights small enough that float16 holds the products of the widest blocks
    x, w = fp8_matrix(m, k, dtype, m + k), fp8_matrix(n, k, torch.float32, n + k, spread=n % 2 == 0) * 2.0 ** -7
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    wq, ws = ops.quantize_fp8(w)
    hq, he = oo.quantize_fp8(oo.host64(w))
    for b, relu in ((bias, True), (None, False)):
        y = ops.matmul_fp8(x, wq, ws, bias=b, relu=relu)
        assert y.dtype == dtype
        ref, bound = oo.matmul_fp8(oo.host64(x), hq, he, None if b is None else oo.host64(b), relu, dtype)
        within(y, ref, bound, "y")
        # all results together: half a step each at most, and a sum's error, which does not add up with one sign
        if m * n >= 64:
            assert np.linalg.norm(oo.host64(y) - ref) <= (oo.HALF_STEP[dtype] + 2.0 ** -13) * np.linalg.norm(ref)
        assert torch.equal(y, ops.matmul_fp8(misaligned(x), wq, ws, bias=b, relu=relu))


@pytest.mark.parametrize("shape", [(1, 17, 33000), (16, 33, 2500), (17, 24577, 640), (40, 24600, 1100)], ids=str)
@pytest.mark.parametrize("dtype", FP8_DTYPES, ids=str)
def test_matmul_fp8_at_the_ends_of_its_operands(ops, shape, dtype):
    """Tiles that hold one row of the weights, or rows of x whose other half is behind the last; words of one to three
    blocks."""
    announce("matmul_fp8 ends", shape, dtype)
    m, n, k = shape
    x, w = fp8_matrix(m, k, dtype, 1), fp8_matrix(n, k, torch.float32, 2) * 2.0 ** -9
    wq, ws = ops.quantize_fp8(w)
    hq, he = oo.quantize_fp8(oo.host64(w))
    ref, bound = oo.matmul_fp8(oo.host64(x), hq, he, None, False, dtype)
    within(ops.matmul_fp8(x, wq, ws), ref, bound, "y")


@pytest.mark.parametrize("m", [3, 60])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("up", [-120, 126])
def test_matmul_fp8_with_scales_at_both_ends(ops, m, dtype, up):
    """Values of one sign and size, whose scales are 2^-127 and 2^118, against weights that bring the product back."""
    announce("matmul_fp8 scales", m, dtype, up)
    g = torch.Generator().manual_seed(m)
    x = ((1 + torch.rand(m, 300, generator=g).double() * 0.9) * 2.0 ** up).to(dtype).cuda()
    w = ((1 + torch.rand(70, 300, generator=g).double() * 0.9) * 2.0 ** (-up * 5 // 6)).float().cuda()
    wq, ws = ops.quantize_fp8(w)
    hq, he = oo.quantize_fp8(oo.host64(w))
    ref, bound = oo.matmul_fp8(oo.host64(x), hq, he, None, False, dtype)
    within(ops.matmul_fp8(x, wq, ws), ref, bound, "y")


def test_matmul_fp8_keeps_what_is_not_a_number_in_its_row(ops):
    announce("matmul_fp8 NaN")
    for m in (5, 200):
        x, w = fp8_matrix(m, 700, torch.float32, 1), fp8_matrix(40, 700, torch.float32, 2)
        wq, ws = ops.quantize_fp8(w)
        clean = ops.matmul_fp8(x, wq, ws)
        x[1, 600], x[3, 0] = float("nan"), float("-inf")
        y = ops.matmul_fp8(x, wq, ws)
        assert torch.isnan(y[[1, 3]]).all()
        rest = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(y[rest], clean[rest])
        w[7, 699] = float("inf")
        y = ops.matmul_fp8(fp8_matrix(m, 700, torch.float32, 1), *ops.quantize_fp8(w))
        assert torch.isnan(y[:, 7]).all() and torch.equal(y[:, :7], clean[:, :7]) and torch.equal(y[:, 8:], clean[:, 8:])


def test_matmul_fp8_of_strided_rows_and_of_none(ops):
    announce("matmul_fp8 strides")
    x, w = fp8_matrix(24, 400, torch.bfloat16, 3), fp8_matrix(40, 200, torch.float32, 4)
    wq, ws = ops.quantize_fp8(w)
    assert torch.equal(ops.matmul_fp8(x[:, ::2], wq, ws), ops.matmul_fp8(x[:, ::2].contiguous(), wq, ws))
    assert ops.matmul_fp8(x[:0, :200], wq, ws).shape == (0, 40)
    with pytest.raises(ValueError):
        ops.matmul_fp8(x[:, :200], wq.as_strided(wq.shape, (1, 40)), ws)


def test_matmul_fp8_in_graphs_and_on_two_streams(ops):
    announce("matmul_fp8 graphs")
    cases = []
    for m, n, k in ((16, 300, 9000), (3, 1000, 4096), (400, 300, 1000)):
        x, w = fp8_matrix(m, k, torch.float32, m), fp8_matrix(n, k, torch.float32, n)
        wq, ws = ops.quantize_fp8(w)
        cases.append((x, wq, ws, ops.matmul_fp8(x, wq, ws, relu=True)))
    torch.cuda.synchronize()
    graphs = []
    for x, wq, ws, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.matmul_fp8(x, wq, ws, relu=True)))
        graphs[-1] = (graph, graphs[-1][1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, y in graphs:
            y.zero_()
        torch.cuda.synchronize()
        eager = []
        for stream, (graph, y), (x, wq, ws, ref) in zip(streams, graphs, cases):
            with torch.cuda.stream(stream):
                graph.replay()
                eager.append(ops.matmul_fp8(x, wq, ws, relu=True))
        torch.cuda.synchronize()
        for (graph, y), e, (x, wq, ws, ref) in zip(graphs, eager, cases):
            assert torch.equal(y, ref) and torch.equal(e, ref)


# --------------------------------------------------------------------------- layers
@pytest.mark.parametrize("fmt", ["NCHW", "NHWC"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
def test_group_normalization_layer(pd, fmt, dtype):
    announce("group normalization layer", fmt, dtype)
    nhwc = fmt == "NHWC"
    model = pd.Model(dtype=dtype, tensor_format=fmt)
    model.mode = pd.TRAIN_MODE
    layer = pd.GroupNormalization(groups=4, gamma=1.5, beta=-0.25, activation="relu")
    layer.set_model(model)
    shape = (6, 7, 24) if nhwc else (24, 6, 7)
    layer.initialize(shape)
    assert layer.shape == shape and layer.nparams == 48
    x, dy, _, _, _ = gn_inputs((3, (6, 7), 24, 4), dtype, nhwc, 26)
    y, dx = layer.forward(x), layer.backward(dy)
    hx, hdy, hg, hb = (oo.host64(t) for t in (x, dy, layer.gamma, layer.beta))
    ref = oo.gn_forward(hx, hg, hb, 4, 1e-5, "relu", nhwc)
    within(y, ref[0], oo.gn_forward_bounds(hx, hg, hb, 4, 1e-5, nhwc, ref[0], dtype)[0], "y")
    hm, hi = oo.host64(layer.mean), oo.host64(layer.inv_std)
    ref = oo.gn_backward(hdy, hx, hg, hb, hm, hi, 4, "relu", nhwc)
    bounds = oo.gn_backward_bounds(hdy, hx, hg, hb, hm, hi, 4, "relu", nhwc, ref[2], dtype)
    for got, r, b, what in zip((layer.dgamma, layer.dbeta, dx), ref, bounds, ("dgamma", "dbeta", "dx")):
        within(got, r, b, what)
    model.mode = pd.EVALUATE_MODE
    assert torch.equal(layer.forward(x), y)
    with pytest.raises(ValueError):
        other = pd.GroupNormalization(groups=5)
        other.set_model(model)
        other.initialize(shape)


def test_dropout_layer_with_a_seed(pd):
    announce("dropout layer")
    model = pd.Model()
    model.mode = pd.TRAIN_MODE
    layers = [pd.Dropout(rate=0.25, seed=99), pd.Dropout(rate=0.25, seed=99)]
    for layer in layers:
        layer.set_model(model)
        layer.initialize((50,))
    x = torch.randn(8, 50, device="cuda")
    masks = []
    for step in (1, 2):
        for layer in layers:
            y = layer.forward(x)
            assert torch.equal(y.cpu(), oo.dropout(x, 0.25, 99 + (layer.id << 32), step))
            assert torch.equal(layer.backward(x), y) and layer.mask is None
            masks.append(y != 0)
    assert not any(torch.equal(masks[i], masks[j]) for i in range(4) for j in range(i))
    layers[0].step.fill_(0)
    assert torch.equal(layers[0].forward(x) != 0, masks[0])
    model.mode = pd.EVALUATE_MODE
    assert layers[0].forward(x) is x and layers[0].backward(x) is x


def test_fc_in_8_bits_after_the_fusion_pass(pd):
    announce("FC in 8 bits")
    rng = np.random.default_rng(4)
    model = pd.Model(enable_fp8_fc=True)
    model.add(pd.Input(shape=(300,)))
    model.add(pd.FC(shape=(70,), activation="relu"))
    model.add(pd.FC(shape=(10,), use_bias=False, activation="softmax"))
    model.layers[1].biases = torch.from_numpy(rng.standard_normal(70).astype(np.float32)).cuda()
    stored = {}
    model.load_store_path(model.layers, stored, "store")
    x = torch.randn(9, 300, device="cuda")
    y = model.evaluate_dataset_batch(x)
    assert [type(layer).__name__ for layer in model.layers] == ["Input", "FCFp8", "FCFp8", "Softmax"]
    cur = x
    for layer in model.layers[1:3]:
        out = layer.forward(cur)
        hq, he = oo.quantize_fp8(oo.host64(layer.weights).T)
        ref, bound = oo.matmul_fp8(oo.host64(cur), hq, he, oo.host64(layer.biases) if layer.use_bias else None, layer.relu,
                                   torch.float32)
        within(out, ref, bound, "FC")
        cur = out
    assert model.layers[1].relu and not model.layers[2].relu
    assert torch.equal(model.layers[3].forward(cur), y)
    again = {}
    model.load_store_path(model.layers, again, "store")
    assert sorted(again) == sorted(stored) and all(np.array_equal(again[k], stored[k]) for k in stored)
    # weights that are loaded are quantised anew
    model.load_store_path(model.layers, {k: v * 2 for k, v in stored.items()}, "load")
    assert torch.equal(model.layers[2].forward(model.layers[1].forward(x)), 4 * cur)
    with pytest.raises(RuntimeError):
        model.train_batch(x, y, pd.CategoricalCrossEntropy(), pd.SGD())
    with pytest.raises(RuntimeError):
        model.layers[1].backward(y)


@pytest.mark.parametrize("fmt", ["NCHW", "NHWC"])
def test_a_network_is_trained_with_group_norm_and_dropout_and_served_in_8_bits(pd, fmt):
    """One step of a network whose blocks are normalised by groups and whose head drops by a seed, against the same network
    in float64 on the CPU with the oracle's masks and torch's gradients, and the network served in 8 bits afterwards."""
    announce("network", fmt)
    nhwc = fmt == "NHWC"
    model = pd.Model(tensor_format=fmt, enable_fp8_fc=True)
    model.add(pd.Input(shape=(12, 10, 3)))
    model.add(pd.Conv2D(nfilters=16, filter_shape=(3, 3), padding=1, use_bias=False))      # 1
    model.add(pd.GroupNormalization(groups=4, activation="silu"))                           # 2
    model.add(pd.MaxPool2D(pool_shape=(2, 2), stride=2))                                    # 3
    model.add(pd.Conv2D(nfilters=24, filter_shape=(3, 3), padding=1, use_bias=False))      # 4
    model.add(pd.GroupNormalization(groups=8))                                              # 5
    model.add(pd.Flatten())                                                                 # 6
    model.add(pd.FC(shape=(40,)))                                                           # 7
    model.add(pd.Dropout(rate=0.5, seed=31))                                                # 8
    model.add(pd.FC(shape=(10,), activation="softmax"))                                     # 9, 10
    g = torch.Generator().manual_seed(2)
    x = torch.randn((6, 12, 10, 3) if nhwc else (6, 3, 12, 10), generator=g)
    labels = torch.randint(0, 10, (6,), generator=g)
    target = torch.zeros(6, 10)
    target[torch.arange(6), labels] = 1
    layers = model.layers
    names = [(i, v) for i in (1, 2, 4, 5, 7, 9) for v in layers[i].grad_vars]
    before = {(i, v): getattr(layers[i], v).double().cpu().clone().requires_grad_() for i, v in names}
    loss = model.train_batch(x.cuda(), target.cuda(), pd.CategoricalCrossEntropy(), pd.SGD(learning_rate=0.0))

    def conv(t, w):
        w = w.permute(3, 0, 1, 2) if nhwc else w
        t = t.permute(0, 3, 1, 2) if nhwc else t
        t = torch.nn.functional.conv2d(t, w, padding=1)
        return t.permute(0, 2, 3, 1) if nhwc else t

    def norm(t, i, groups):
        t = t.permute(0, 3, 1, 2) if nhwc else t
        t = torch.nn.functional.group_norm(t, groups, before[i, "gamma"], before[i, "beta"], 1e-5)
        return t.permute(0, 2, 3, 1) if nhwc else t

    t = torch.nn.functional.silu(norm(conv(x.double(), before[1, "weights"]), 2, 4))
    t = torch.nn.functional.max_pool2d(t.permute(0, 3, 1, 2), 2).permute(0, 2, 3, 1) if nhwc else \
        torch.nn.functional.max_pool2d(t, 2)
    t = norm(conv(t, before[4, "weights"]), 5, 8).reshape(6, -1)
    t = t @ before[7, "weights"] + before[7, "biases"]
    t = t * oo.dropout(torch.ones(6, 40, dtype=torch.float64), 0.5, 31 + (layers[8].id << 32), 1)
    t = t @ before[9, "weights"] + before[9, "biases"]
    ref = torch.nn.functional.cross_entropy(t, labels)
    ref.backward()
    # float32 through nine layers: each a sum of at most 720 terms, far from cancelling, so a part in 10^4 of the
    # largest gradient is over a thousand half steps
    assert abs(float(loss) - float(ref)) < 1e-4 * float(ref)
    for i, v in names:
        got, want = getattr(layers[i], layers[i].grad_vars[v]).double().cpu(), before[i, v].grad
        assert got.reshape(want.shape).sub(want).abs().max() < 1e-4 * want.abs().max(), (i, v)
    plain = model.evaluate_batch(x.cuda())
    served = model.evaluate_dataset_batch(x.cuda())
    assert type(model.layers[7]).__name__ == type(model.layers[9]).__name__ == "FCFp8"
    cur = x.cuda()
    for layer in model.layers[1:]:
        out = layer.forward(cur)
        if type(layer).__name__ == "FCFp8":
            hq, he = oo.quantize_fp8(oo.host64(layer.weights).T)
            want, bound = oo.matmul_fp8(oo.host64(cur), hq, he, oo.host64(layer.biases), False, torch.float32)
            within(out, want, bound, "FC")
        cur = out
    assert torch.equal(cur, served) and served.shape == plain.shape


def test_builders_with_group_norm_and_seeded_dropout(pd):
    announce("builders")
    model = pd.Model(tensor_format="NHWC")
    pd.models.create_resnet50_imagenet(model, stages=((16, 1, 1), (32, 1, 2)), classes=7, input_shape=(32, 32, 3), groups=4)
    kinds = {type(layer).__name__ for layer in model.get_all_layers()}
    assert "GroupNormalization" in kinds and "BatchNormalization" not in kinds
    x = torch.randn(2, 32, 32, 3, device="cuda")
    target = torch.eye(7, device="cuda")[:2].contiguous()
    loss = model.train_batch(x, target, pd.CategoricalCrossEntropy(), pd.SGD())
    assert torch.isfinite(loss)
    for layer in model.get_all_layers():
        if type(layer).__name__ == "GroupNormalization":
            assert torch.isfinite(layer.dgamma).all() and layer.dgamma.abs().max() > 0


# --------------------------------------------------------------------------- sums of the e4m3 product
@pytest.mark.parametrize("m", [2, 40])
@pytest.mark.parametrize("dtype", FP8_DTYPES, ids=str)
def test_matmul_fp8_adds_what_its_documentation_says(ops, m, dtype):
    """Two eights whose largest products, 2^16 and -2^16, cancel and leave seven products of 2^3 and seven of 2^2: the former
    are 13 bits below the largest, the latter 14.  In 24 bits the sum is 84; for 16-bit types it is off by at most 7 * 2^-13 of
    the largest product of each eight, which is what the test's bound is of."""
    announce("matmul_fp8 cancelling", m, dtype)
    row = torch.zeros(128)
    row[0], row[8] = 256.0, -256.0
    row[1:8], row[9:16] = 2.0, 1.0
    weights = torch.zeros(128)
    weights[0] = weights[8] = 256.0
    weights[1:8] = weights[9:16] = 4.0
    x = row.repeat(m, 1).to(dtype).cuda()
    wq, ws = ops.quantize_fp8(weights.repeat(20, 1).cuda())
    y = oo.host64(ops.matmul_fp8(x, wq, ws))
    if dtype == torch.float32:
        assert np.all(y == 84.0)
    else:
        assert np.all(np.abs(y - 84.0) <= 2 * 7 * 2.0 ** -13 * 2.0 ** 16)
        assert torch.all(ops.matmul_fp8(x.float(), wq, ws) == 84.0)
    ref, bound = oo.matmul_fp8(oo.host64(x), *oo.quantize_fp8(oo.host64(weights.repeat(20, 1))), None, False, dtype)
    assert np.all(ref == 84.0) and np.all(np.abs(y - ref) <= bound)


# --------------------------------------------------------------------------- group norm: few images of many runs
def least_us(f):
    """The least time of a call among calls, of five blocks of ten."""
    f()
    torch.cuda.synchronize()
    times = []
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(10):
            f()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end) * 100)
    return min(times)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, (90, 88), 520, 520), (1, (112, 112), 256, 1), (2, (61, 60), 512, 128), (1, (120, 121), 27, 9)],
                         ids=str)
def test_group_norm_of_few_images_of_many_runs(ops, shape, dtype):
    """Images cut into hundreds of runs, whose sums kernels of their own join."""
    announce("group norm, many runs", shape, dtype)
    x, dy, gamma, beta, groups = gn_inputs(shape, dtype, True, 8)
    check_gn(ops, x, dy, gamma, beta, groups, "silu", True)
    check_gn(ops, misaligned(x), dy, gamma, beta, groups, "relu", True)


@pytest.mark.parametrize("groups", [1, 16, 64, 256, 1024])
def test_group_norm_of_one_large_image_costs_a_few_copies(ops, groups):
    """What the second pass joins does not grow with the square of the runs: one image of 51 MB, cut into over 700 runs, takes
    at most eight times what a copy of it takes in either direction (they move it three and five times)."""
    announce("group norm, one image", groups)
    x, dy, gamma, beta, _ = gn_inputs((1, (112, 112), 1024, groups), torch.float32, True, 9)
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups)
    copy = least_us(x.clone)
    forward = least_us(lambda: ops.gn_forward(x, gamma, beta, groups))
    backward = least_us(lambda: ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups))
    print(f"copy {copy:.1f} us, forward {forward:.1f}, backward {backward:.1f}")
    assert forward < 8 * copy and backward < 8 * copy, (copy, forward, backward)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(3, (7, 7), 2049, 1), (2, (14, 14), 1026, 1), (2, (3, 3), 18000, 2), (1, (33, 31), 600, 1)], ids=str)
def test_group_norm_of_groups_of_many_planes(ops, shape, dtype):
    """Groups of more planes than a workgroup holds, whose moments a kernel of its own joins."""
    announce("group norm, many planes", shape, dtype)
    x, dy, gamma, beta, groups = gn_inputs(shape, dtype, False, 8)
    check_gn(ops, x, dy, gamma, beta, groups, "silu", False)
    check_gn(ops, misaligned(x), dy, gamma, beta, groups, "relu", False)


def test_group_norm_of_many_small_planes_costs_a_few_copies(ops):
    """What the planes of a group join does not grow with the square of their number: 131072 planes of 7 x 7 in one group an
    image, 25.7 MB, take at most fifteen times what a copy takes (forward moves them three times, and each of its three launches
    takes as long as a copy of this size)."""
    announce("group norm, small planes")
    x, _, gamma, beta, _ = gn_inputs((64, (7, 7), 2048, 1), torch.float32, False, 9)
    copy = least_us(x.clone)
    forward = least_us(lambda: ops.gn_forward(x, gamma, beta, 1, nhwc=False))
    print(f"copy {copy:.1f} us, forward {forward:.1f}")
    assert forward < 15 * copy, (copy, forward)


# --------------------------------------------------------------------------- group norm: tensors too large for the host form
def of_group(t, nhwc, images, channels):
    return t[images][..., channels] if nhwc else t[images][:, channels]


def check_gn_of_groups(ops, x, dy, gamma, beta, groups, activation, nhwc, samples, eps=1e-5):
    """check_gn for a few (image, group): y, the statistics and dx of each against the 64-bit form of that group by itself,
    dgamma and dbeta of its channels against sums in 64 bits over all images."""
    dtype, cg = x.dtype, gamma.numel() // groups
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, eps, activation, nhwc)
    dgamma, dbeta, dx = ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, activation, nhwc)
    for image, group in samples:
        at, ch = slice(image, image + 1), slice(group * cg, (group + 1) * cg)
        hx, hdy, hg, hb = (oo.host64(t) for t in (of_group(x, nhwc, at, ch), of_group(dy, nhwc, at, ch), gamma[ch], beta[ch]))
        ref = oo.gn_forward(hx, hg, hb, 1, eps, activation, nhwc)
        bounds = oo.gn_forward_bounds(hx, hg, hb, 1, eps, nhwc, ref[0], dtype)
        got = (of_group(y, nhwc, at, ch), mean[at, group:group + 1], inv_std[at, group:group + 1])
        for g, r, b, what in zip(got, ref, bounds, ("y", "mean", "inv_std")):
            within(g, r, b, (what, image, group))
        hm, hi = oo.host64(got[1]), oo.host64(got[2])
        ref = oo.gn_backward(hdy, hx, hg, hb, hm, hi, 1, activation, nhwc)[2]
        bound = oo.gn_backward_bounds(hdy, hx, hg, hb, hm, hi, 1, activation, nhwc, ref, dtype)[2]
        within(of_group(dx, nhwc, at, ch), ref, bound, ("dx", image, group))
    for group in sorted({g for _, g in samples}):
        ch = slice(group * cg, (group + 1) * cg)
        sums = torch.zeros(4, cg, dtype=torch.float64, device=x.device)      # dz xn, dz and the magnitudes of each
        for i in range(x.shape[0]):
            xi, di = (of_group(t, nhwc, slice(i, i + 1), ch).double() for t in (x, dy))
            if not nhwc:
                xi, di = xi.transpose(1, -1), di.transpose(1, -1)
            xi, di = xi.reshape(-1, cg), di.reshape(-1, cg)
            xn = (xi - mean[i, group].double()) * inv_std[i, group].double()
            z = xn * gamma[ch].double() + beta[ch].double()
            dz = di * (z > 0) if activation == "relu" else di
            sums += torch.stack([(dz * xn).sum(0), dz.sum(0), (dz * xn).abs().sum(0), dz.abs().sum(0)])
        # as in gn_backward_bounds
        u, n = oo.WIDE_HALF_STEP[dtype], x.numel() // gamma.numel()
        k = (8 * n ** 0.5 + 8) * u
        ref = oo.host64(sums)
        within(dgamma[ch], ref[0], (k + 7 * u) * ref[2], ("dgamma", group))
        within(dbeta[ch], ref[1], k * ref[3], ("dbeta", group))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
@pytest.mark.parametrize("images,pixels", [(64, (7, 7)), (500, (14, 14))])
def test_group_norm_of_a_slab_that_leaves_threads_idle(ops, images, pixels, dtype):
    """17 groups: one kernel holds a slab of a group, and no wider one fits."""
    announce("group norm, idle slab", images, pixels, dtype)
    c = 544 if dtype == torch.float32 else 272
    x, dy, gamma, beta, groups = gn_inputs((images, pixels, c, 17), dtype, True, 3)
    check_gn_of_groups(ops, x, dy, gamma, beta, groups, "relu", True, [(0, 0), (images // 2, 7), (images - 1, 16)])


@pytest.mark.parametrize("activation", ["", "relu"])
@pytest.mark.parametrize("nhwc", [True, False], ids=["last", "first"])
def test_group_norm_of_more_than_2_to_31_elements_in_64_bits(ops, nhwc, activation):
    """Groups of the first image and of the last, whose elements lie beyond 2^31, in either format; 32 channels and 2^18 pixels
    a group."""
    announce("group norm beyond 32 bits in 64 bits", nhwc, activation)
    images, pixels, c, groups = 9, 1 << 18, 1024, 32
    shape = (images, pixels, c) if nhwc else (images, c, pixels)
    x, dy = (torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for i in range(images):
        g = torch.Generator(device="cuda").manual_seed(i)
        x[i].normal_(mean=0.5, std=1.5, generator=g)
        dy[i].normal_(generator=g)
    gamma, beta = torch.rand(c, device="cuda") + 0.5, torch.randn(c, device="cuda")
    check_gn_of_groups(ops, x, dy, gamma, beta, groups, activation, nhwc, [(0, 0), (8, 31)])


# --------------------------------------------------------------------------- the larger tiles of the e4m3 product
# (m, n, k) that take tiles of 256 (16-bit types; at least 192 of them) and of 128, several in each direction, ragged in every
# extent, the last bands of tiles partly empty
FP8_TILES = [(3000, 4099, 300), (2900, 4200, 1100), (4100, 2900, 129), (1500, 2100, 700), (2060, 1540, 1), (1800, 1795, 2050)]


@pytest.mark.parametrize("dtype", FP8_DTYPES, ids=str)
@pytest.mark.parametrize("shape", FP8_TILES, ids=str)
def test_matmul_fp8_in_the_larger_tiles(ops, shape, dtype):
    m, n, k = shape
    announce("matmul_fp8, larger tiles", shape, dtype)
    x, w = fp8_matrix(m, k, dtype, m + k), fp8_matrix(n, k, torch.float32, n + k) * 2.0 ** -7
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    wq, ws = ops.quantize_fp8(w)
    hq, he = oo.quantize_fp8(oo.host64(w))
    y = ops.matmul_fp8(x, wq, ws, bias=bias, relu=True)
    plain = ops.matmul_fp8(misaligned(x), wq, ws)
    # rows of every tile and the ragged ends, all columns
    rows = sorted({*range(0, m, 37), *range(0, m, 64), *range(63, m, 64), *range(max(0, m - 20), m)})
    hx, hy = oo.host64(x[rows]), oo.host64(y[rows])
    ref, bound = oo.matmul_fp8(hx, hq, he, oo.host64(bias), True, dtype)
    within(y[rows], ref, bound, "y")
    assert np.linalg.norm(hy - ref) <= (oo.HALF_STEP[dtype] + 2.0 ** -13) * np.linalg.norm(ref)
    ref, bound = oo.matmul_fp8(hx, hq, he, None, False, dtype)
    within(plain[rows], ref, bound, "y without bias")
    # every other row: as the same rows in another order, which puts them in other places of other tiles
    order = torch.randperm(m, generator=torch.Generator().manual_seed(k)).cuda()
    assert torch.equal(ops.matmul_fp8(x[order], wq, ws, bias=bias, relu=True), y[order])


@pytest.mark.parametrize("shape", [(131100, 16, 16400), (50001, 43003, 128), (3, 131100, 16400), (40, 131100, 16400)], ids=str)
def test_matmul_fp8_of_more_than_2_to_31_elements(ops, shape):
    """Activations, results and weights (for a few rows and for more) beyond 2^31 elements: their first and last rows."""
    m, n, k = shape
    announce("matmul_fp8 beyond 32 bits", shape)
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.empty((n, k), dtype=torch.bfloat16, device="cuda").normal_(std=2.0 ** -7, generator=g)
    y = ops.matmul_fp8(x, *ops.quantize_fp8(w))
    rows = sorted({0, 1, m // 2, *range(max(0, m - 12), m)} & set(range(m)))
    columns = sorted({0, 1, n // 2, *range(max(0, n - 20), n)} & set(range(n)))
    hq, he = oo.quantize_fp8(oo.host64(w[columns]))
    ref, bound = oo.matmul_fp8(oo.host64(x[rows]), hq, he, None, False, torch.bfloat16)
    within(y[rows][:, columns], ref, bound, "y")


def test_group_norm_silu_is_as_exact_as_its_documentation_says(ops):
    """Constant groups, whose z is the shift itself: 1 / (1 + exp(-z)) within (3 + |z|) steps of 2^-23 (the hardware's 2^v and
    1/v a step each, the sum half a step, the exponent's rounding 0.63 |z| of a step), one more half step for the product, and 0
    under -126 log 2, where 1 + exp(-z) is over 2^126 and its reciprocal below the smallest normal number; its derivative
    p (1 + z (1 - p)) with p off by as much and three roundings of (1 + |z|)."""
    announce("group norm silu")
    z = np.concatenate([np.linspace(-87.3, 88.7, 6001), np.linspace(-3, 3, 2001), [-1e4, -200.0, -104.0, -88.0, -87.5, 200.0, 1e4],
                        [0.0, 2.0 ** -60, -2.0 ** -60, 2.0 ** -140]])
    beta = torch.from_numpy(z).float().cuda()
    z = oo.host64(beta)
    c = len(z)
    x, gamma = torch.full((1, 1, c), 2.5, device="cuda"), torch.ones(c, device="cuda")
    y, mean, inv_std = ops.gn_forward(x, gamma, beta, c, 1e-5, "silu")
    with np.errstate(over="ignore"):
        p = 1 / (1 + np.exp(-z))
    e = (3 + np.abs(z)) * 2.0 ** -23
    low = z < -126 * np.log(2)      # -87.3365
    got = oo.host64(y).reshape(-1)
    assert np.all(got[low] == 0)
    assert np.all(np.abs(got - z * p)[~low] <= ((e + 2.0 ** -24) * np.abs(z * p) + 2.0 ** -149)[~low])
    dbeta = oo.host64(ops.gn_backward(torch.ones_like(x), x, gamma, beta, mean, inv_std, c, "silu")[1])
    bound = p * (e * np.abs(1 + z * (1 - p)) + np.abs(z) * p * e + (1 + np.abs(z)) * 2.0 ** -22) + 2.0 ** -149
    assert np.all(np.abs(dbeta - p * (1 + z * (1 - p)))[~low] <= bound[~low]) and np.all(dbeta[low] == 0)


def test_group_norm_whose_sums_are_joined_once_in_graphs_and_on_two_streams(ops):
    """The forms with kernels between their two passes, captured, replayed and called at once."""
    announce("group norm joined, graphs and streams")
    cases = [(gn_inputs((1, (90, 88), 520, 520), torch.float32, True, 31), True),
             (gn_inputs((3, (7, 7), 2049, 1), torch.float32, False, 32), False)]

    def both(case, nhwc):
        x, dy, gamma, beta, groups = case
        y, mean, inv_std = ops.gn_forward(x, gamma, beta, groups, activation="relu", nhwc=nhwc)
        return (y, mean, inv_std, *ops.gn_backward(dy, x, gamma, beta, mean, inv_std, groups, "relu", nhwc))

    eager = [both(*case) for case in cases]
    torch.cuda.synchronize()
    graphs = []
    for case in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(*case)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for _, out in graphs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        again = []
        for stream, (graph, _), case in zip(streams, graphs, cases):
            with torch.cuda.stream(stream):
                graph.replay()
                again.append(both(*case))
        torch.cuda.synchronize()
        for (_, out), now, ref in zip(graphs, again, eager):
            assert all(torch.equal(t, r) for t, r in zip(out, ref)) and all(torch.equal(t, r) for t, r in zip(now, ref))
