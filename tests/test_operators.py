"""CPU-side checks of the operators for several element types: the oracles against published values and differences, and
what the entry points refuse (nothing here launches a kernel)."""
import ctypes
import inspect
import os

import numpy as np
import pytest
import torch

import operator_oracles as oo


@pytest.fixture(scope="module")
def lib():
    from pydtnn_amd import native
    if not os.path.exists(native.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return native.lib()


@pytest.fixture(scope="module")
def ops(lib):
    from pydtnn_amd import ops
    return ops


@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_the_generator_gives_its_authors_known_answers(counter, key, words):
    """The known answers that the authors of Philox4x32-10 publish for it."""
    assert tuple(int(w[0]) for w in oo.philox4x32_10([[c] for c in counter], key)) == words


@pytest.mark.parametrize("activation", ["", "silu"])
@pytest.mark.parametrize("nhwc", [True, False])
def test_the_group_norm_gradient_of_the_oracle_is_the_slope_of_its_forward(activation, nhwc):
    rng = np.random.default_rng(3)
    shape = (2, 3, 4, 6) if nhwc else (2, 6, 3, 4)
    x, dy = rng.standard_normal(shape), rng.standard_normal(shape)
    gamma, beta = rng.standard_normal(6), rng.standard_normal(6)

    def loss(x, gamma, beta):
        return (oo.gn_forward(x, gamma, beta, 3, 1e-5, activation, nhwc)[0] * dy).sum()

    _, mean, inv_std = oo.gn_forward(x, gamma, beta, 3, 1e-5, activation, nhwc)
    grads = oo.gn_backward(dy, x, gamma, beta, mean, inv_std, 3, activation, nhwc)
    h = 1e-5
    for which, grad in ((1, grads[0]), (2, grads[1]), (0, grads[2])):
        for _ in range(4):
            v = [np.zeros(shape), np.zeros(6), np.zeros(6)]
            v[which] = rng.standard_normal(v[which].shape)
            slope = (loss(x + h * v[0], gamma + h * v[1], beta + h * v[2]) -
                     loss(x - h * v[0], gamma - h * v[1], beta - h * v[2])) / (2 * h)
            # the third derivative's h^2 and the difference's rounding, 1e-16 |loss| / h
            assert abs(slope - (grad * v[which]).sum()) < 1e-6


FAKE = 4096      # an address that a call which refuses its arguments never touches


def test_gn_refuses_extents_it_cannot_run(lib):
    p = ctypes.c_void_p(FAKE)

    def forward(dtype=0, images=2, channels=8, pixels=4, groups=2, eps=1e-5, act=0, x=p, nbytes=None):
        need = lib.pydtnn_hip_gn_workspace_bytes(dtype, 0, 0, images, channels, pixels, groups, 1)
        return lib.pydtnn_hip_gn_forward(dtype, 0, x, p, p, p, p, p, images, channels, pixels, groups, eps, act, p,
                                         need - 1 if nbytes else need, None)

    assert forward(x=None) == 1
    assert forward(images=0) == forward(pixels=0) == forward(channels=0) == forward(groups=0) == 1
    assert forward(groups=3) == 1
    assert forward(eps=-1.0) == forward(eps=float("nan")) == 1
    assert forward(pixels=1 << 20, nbytes=-1) == 2          # (what a workgroup's registers hold needs none)
    assert forward(dtype=9) in (1, 2) and forward(act=7) == 1
    assert forward(pixels=(1 << 30) + 1) == 4
    assert lib.pydtnn_hip_gn_backward(0, 1, p, p, p, p, p, p, p, None, p, 2, 8, 4, 2, 0, p, 1 << 20, None) == 1
    assert lib.pydtnn_hip_gn_backward(0, 1, p, p, p, p, p, p, p, p, p, 2, 8, 4, 2, 0, p, 8, None) == 2


@pytest.mark.parametrize("nhwc", [0, 1])
def test_gn_refuses_launches_of_too_many_threads(lib, nhwc):
    """Images of one pixel of very many channels, in groups of one: the kernels of the channels and of the groups would have
    2^32 threads and more.  (The workspace is never touched.)"""
    p = ctypes.c_void_p(FAKE)
    for images, channels in ((1, 1 << 26), (1, 1 << 30), (1 << 12, 1 << 14)):
        need = lib.pydtnn_hip_gn_workspace_bytes(0, nhwc, 1, images, channels, 1, channels, 1)
        if nhwc and channels == 1 << 14:
            continue                                      # (runs)
        assert lib.pydtnn_hip_gn_backward(0, nhwc, p, p, p, p, p, p, p, p, p, images, channels, 1, channels, 0, p, need,
                                          None) == 4


def test_dropout_refuses_rates_and_types_it_does_not_know(lib):
    p = ctypes.c_void_p(FAKE)
    for rate in (-0.1, 1.1, float("nan")):
        assert lib.pydtnn_hip_dropout(0, p, p, 8, rate, 1, 0, None, None) == 1
    assert lib.pydtnn_hip_dropout(4, p, p, 8, 0.5, 1, 0, None, None) == 1
    assert lib.pydtnn_hip_dropout(0, p, p, 0, 0.5, 1, 0, None, None) == 1
    assert lib.pydtnn_hip_dropout(0, None, p, 8, 0.5, 1, 0, None, None) == 1
    assert lib.pydtnn_hip_dropout(0, p, p, 1 << 45, 0.5, 1, 0, None, None) == 4


def test_gn_checks_its_tensors(ops):
    x, v, s = torch.ones(2, 3, 3, 8), torch.ones(8), torch.ones(2, 4)
    with pytest.raises(ValueError):
        ops.gn_forward(x, v, v, 4)                                  # not on the GPU
    with pytest.raises(ValueError):
        ops.gn_forward(x, v, v, 3)
    with pytest.raises(ValueError):
        ops.gn_forward(x, v, v, 0)
    with pytest.raises(ValueError):
        ops.gn_forward(x, v[:4], v, 4)
    with pytest.raises(ValueError):
        ops.gn_forward(x, v, v, 4, activation="tanh")
    with pytest.raises(ValueError):
        ops.gn_forward(x, v, v, 4, eps=-1e-5)
    with pytest.raises(ValueError):
        ops.gn_forward(v, v, v, 4)
    with pytest.raises(ValueError):
        ops.gn_forward(x[:, :0], v, v, 4)
    with pytest.raises(TypeError):
        ops.gn_forward(x.int(), v, v, 4)
    with pytest.raises(TypeError):
        ops.gn_forward(x.half(), v.half(), v, 4)
    with pytest.raises(TypeError):
        ops.gn_forward(x.double(), v, v, 4)
    with pytest.raises(ValueError):
        ops.gn_backward(x, x, v, v, s[:1], s, 4)
    with pytest.raises(TypeError):
        ops.gn_backward(x.half(), x, v, v, s, s, 4)
    with pytest.raises(ValueError):
        ops.gn_backward(x[:1], x, v, v, s, s, 4)


def test_dropout_checks_its_arguments(ops):
    x = torch.ones(8)
    for rate in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout(x, rate, 1)
    with pytest.raises(ValueError):
        ops.dropout(x, 0.5, 1)                                      # not on the GPU
    with pytest.raises(TypeError):
        ops.dropout(x.int(), 0.5, 1)
    with pytest.raises(TypeError):
        ops.dropout(x, 0.5, 1, torch.zeros(1))
    with pytest.raises(TypeError):
        ops.dropout(x, 0.5, 1, torch.zeros(2, dtype=torch.int64))


def test_a_dropout_layer_checks_its_seed():
    import pydtnn_amd as pd
    for seed in (-1, 1 << 32):
        with pytest.raises(ValueError):
            pd.Dropout(rate=0.5, seed=seed)
    assert pd.Dropout(rate=0.5).seed is None


def test_e4m3_of_the_oracle_is_the_type_of_torch():
    v = np.concatenate([np.linspace(-448, 448, 40001), np.linspace(-0.04, 0.04, 4001), 2.0 ** np.arange(-12, 9.0)])
    v = v.astype(np.float32)
    assert np.array_equal(oo.e4m3(v.astype(np.float64)), oo.host64(torch.from_numpy(v).to(torch.float8_e4m3fn)))


def test_fp8_refuses_what_it_cannot_run(lib):
    p = ctypes.c_void_p(FAKE)

    def quantize(dtype=0, rows=4, k=200, x=p, q=p, s=p):
        return lib.pydtnn_hip_quantize_fp8(dtype, x, rows, k, q, s, None)

    assert quantize(x=None) == quantize(q=None) == quantize(s=None) == 1
    assert quantize(rows=0) == quantize(k=0) == quantize(dtype=1) == quantize(dtype=7) == 1
    assert quantize(q=ctypes.c_void_p(FAKE + 8)) == quantize(s=ctypes.c_void_p(FAKE + 2)) == 1
    assert quantize(k=(1 << 30) + 1) == 4

    def matmul(dtype=0, m=4, k=200, n=6, x=p, w=p, s=p, y=p, ws=p, short=0):
        need = lib.pydtnn_hip_matmul_fp8_workspace_bytes(dtype, m, n, k)
        return lib.pydtnn_hip_matmul_fp8(dtype, x, m, k, w, s, n, None, 0, y, ws, max(need - short, 0), None)

    assert matmul(x=None) == matmul(w=None) == matmul(s=None) == matmul(y=None) == 1
    assert matmul(m=0) == matmul(k=0) == matmul(n=0) == matmul(dtype=1) == 1
    assert matmul(w=ctypes.c_void_p(FAKE + 8)) == 1
    # (a few short rows need no workspace)
    assert lib.pydtnn_hip_matmul_fp8_workspace_bytes(0, 4, 6, 200) == 0
    assert matmul(m=40, ws=None) == matmul(m=40, short=1) == matmul(m=40, ws=ctypes.c_void_p(FAKE + 4)) == 2
    assert matmul(n=(1 << 30) + 1) == 4


def test_fp8_checks_its_tensors(ops):
    x, q, s = torch.ones(3, 200), torch.ones(6, 256).to(torch.float8_e4m3fn), torch.ones(6, 4, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.quantize_fp8(x)                                         # not on the GPU
    with pytest.raises(ValueError):
        ops.matmul_fp8(x, q, s)
    for bad in (x.double(), x.int()):
        with pytest.raises(TypeError):
            ops.quantize_fp8(bad)
        with pytest.raises(TypeError):
            ops.matmul_fp8(bad, q, s)
    for bad in (x[0], x[:, :0], x[None]):
        with pytest.raises(ValueError):
            ops.quantize_fp8(bad)
        with pytest.raises(ValueError):
            ops.matmul_fp8(bad, q, s)
    with pytest.raises(ValueError):
        ops.matmul_fp8(x, q[:, :128], s)
    with pytest.raises(ValueError):
        ops.matmul_fp8(x, q, s[:, :2])
    with pytest.raises(ValueError):
        ops.matmul_fp8(x, q[0], s)
    with pytest.raises(TypeError):
        ops.matmul_fp8(x, q.float(), s)
    with pytest.raises(TypeError):
        ops.matmul_fp8(x, q, s.int())
    with pytest.raises(TypeError):
        ops.matmul_fp8(x, q, s, bias=torch.ones(6).half())
    with pytest.raises(ValueError):
        ops.matmul_fp8(x, q, s, bias=torch.ones(5))


def test_a_float64_model_has_no_8_bit_layers():
    import pydtnn_amd as pd
    with pytest.raises(ValueError):
        pd.Model(dtype="float64", enable_fp8_fc=True)
    with pytest.raises(ValueError):
        pd.Model(dtype="float64").apply_layer_fusion(fp8_fc=True)


def test_fp8_refuses_launches_of_too_many_threads(lib):
    """A wave to each word of four blocks: 2^26 of them would be 2^32 threads."""
    p = ctypes.c_void_p(FAKE)
    for rows, k in ((1 << 26, 128), (1 << 24, 2048), ((1 << 26) - 3, 1)):
        assert lib.pydtnn_hip_quantize_fp8(0, p, rows, k, p, p, None) == 4
        need = lib.pydtnn_hip_matmul_fp8_workspace_bytes(0, rows, 8, k)
        assert lib.pydtnn_hip_matmul_fp8(0, p, rows, k, p, p, 8, None, 0, p, p, need, None) == 4
    assert lib.pydtnn_hip_matmul_fp8(0, p, 1, 128, p, p, 1 << 27, None, 0, p, None, 0, None) == 4


@pytest.mark.parametrize("call", ["gn_forward", "gn_backward", "dropout", "dropout_backward", "quantize_fp8", "matmul_fp8"])
def test_operators_take_their_arguments_by_name(ops, call):
    """Each argument by the name that the signature gives it, the first of them positional or not: the calls get as far as the
    refusal of tensors that are not on the GPU."""
    x, v, s = torch.ones(2, 3, 3, 8), torch.ones(8), torch.ones(2, 4)
    q, scales = torch.ones(6, 256).to(torch.float8_e4m3fn), torch.ones(6, 4, dtype=torch.uint8)
    kwargs = {"gn_forward": dict(x=x, gamma=v, beta=v, groups=4, eps=1e-5, activation="relu", nhwc=True),
              "gn_backward": dict(dy=x, x=x, gamma=v, beta=v, mean=s, inv_std=s, groups=4, activation="", nhwc=True, need_dx=True),
              "dropout": dict(x=x, rate=0.5, seed=1, offset=2),
              "dropout_backward": dict(dy=x, rate=0.5, seed=1, offset=2),
              "quantize_fp8": dict(x=torch.ones(3, 200)),
              "matmul_fp8": dict(x=torch.ones(3, 200), wq=q, wscales=scales, bias=None, relu=True)}[call]
    assert list(inspect.signature(getattr(ops, call)).parameters) == list(kwargs)
    with pytest.raises(ValueError, match="on the GPU"):
        getattr(ops, call)(**kwargs)
    with pytest.raises(ValueError, match="on the GPU"):
        first = next(iter(kwargs))
        getattr(ops, call)(kwargs.pop(first), **kwargs)


@pytest.mark.parametrize("seed", [5, np.int32(5), np.uint32(5), np.uint64(5), np.int64(5)], ids=lambda v: type(v).__name__)
def test_a_dropout_layers_seed_may_be_any_whole_number(seed):
    """The layer's key is seed + (id << 32), which no type of 32 bits holds."""
    import pydtnn_amd as pd
    layer = pd.Dropout(rate=0.5, seed=seed)
    layer.id = 3
    assert layer._key() == 5 + (3 << 32) and type(layer._key()) is int
    for bad in (1.5, "5", np.float32(5)):
        with pytest.raises(TypeError):
            pd.Dropout(rate=0.5, seed=bad)


def test_gn_holds_a_slab_that_fits_where_no_wider_one_does(lib):
    """17 and 19 groups have no divisor to make wider slabs of: forward in one kernel, which needs no workspace."""
    for images, channels, pixels, groups in ((64, 544, 49, 17), (64, 608, 16, 19), (1024, 544, 196, 17)):
        assert lib.pydtnn_hip_gn_workspace_bytes(0, 1, 0, images, channels, pixels, groups, 1) == 0
    # many workgroups of a few idle packs are slower than two passes
    assert lib.pydtnn_hip_gn_workspace_bytes(0, 1, 0, 1024, 544, 49, 17, 1) > 0


def test_dropout_refuses_a_launch_of_too_many_threads(lib):
    p = ctypes.c_void_p(FAKE)
    assert lib.pydtnn_hip_dropout(3, p, p, (1 << 35) - (1 << 11) + 1, 0.5, 1, 0, None, None) == 4
