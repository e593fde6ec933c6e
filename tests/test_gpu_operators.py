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
