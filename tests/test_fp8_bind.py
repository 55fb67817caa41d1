"""What the 8-bit floating-point entries make of their tensors: the arguments that reach the C ABI, caught by a stand-in
of it, so that no GPU is needed."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

import cormorant_b200 as cm
from cormorant_b200 import _lib, kernels

ENTRIES = {
    "cm_quant_fp8": "x x_type q scale rows cols batch ldx ldq lds x_bs q_bs s_bs fmt block_rows",
    "cm_rmsnorm_fp8": "x resid weight resid_out y q scale rows cols ldx ldr ldo ldy ldq lds type weight_type eps fmt",
    "cm_matmul_fp8": "a a_scale b b_scale c n k m lda a_lds ldb b_lds ldc a_fmt b_fmt c_type",
    "cm_matmul_fp8_grouped": "a a_scale b b_scale c offsets groups n k m lda a_lds ldb b_lds b_gs bs_gs ldc a_fmt b_fmt c_type",
}


class OnDevice:
    """A CPU tensor that says it is of cuda:0."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def bytes_(*shape):
    return zeros(*shape, dtype=torch.uint8)


def floats(*shape):
    return zeros(*shape, dtype=torch.float32)


@pytest.fixture
def call():
    """call(entry of kernels.py, arguments) -> what the C ABI was given, by name."""
    seen, keep = [], []

    def stand_in(name, result):
        _, argtypes = _lib.SIGNATURES[name]
        names = ENTRIES.get(name.removesuffix("_async"), "").split()

        def f(*args):
            if names:
                seen.append(SimpleNamespace(entry=name, **dict(zip(names, args))))
            return result

        keep.append(C.CFUNCTYPE(C.c_int, *argtypes)(f))
        return C.cast(keep[-1], C.c_void_p).value

    native = kernels._native()
    native.setup(stand_in("cm_device", 0), *(stand_in(n + t, 0) for n in ENTRIES for t in ("", "_async")))

    def run(entry, *args, **more):
        seen.clear()
        on = lambda v: OnDevice(v) if isinstance(v, torch.Tensor) else v  # noqa: E731
        entry(*map(on, args), **{k: on(v) for k, v in more.items()})
        return seen[0]

    yield run
    kernels._native_module = None            # the library's own addresses again
    kernels._native()


# ---- a pitch that is given leaves the tensor its batch stride -----------------------------------------
@pytest.mark.parametrize("given", [{}, {"ldx": 128}, {"ldq": 144}, {"lds": 133}, {"ldx": 128, "ldq": 144, "lds": 133}])
def test_batch_strides_of_padded_tensors(call, given):
    batch, rows, cols = 3, 130, 100
    x, q, s = zeros(batch, 256, 128)[:, :rows, :cols], bytes_(batch, 200, 144)[:, :rows, :cols], floats(batch, 4, 133)[:, :1, :rows]
    got = call(cm.QuantKernelFp8, x, q, s, rows, cols, batch, **given)
    assert (got.ldx, got.ldq, got.lds) == (128, 144, 133)
    assert (got.x_bs, got.q_bs, got.s_bs) == (256 * 128, 200 * 144, 4 * 133)
    assert (got.x, got.q, got.scale) == (x.data_ptr(), q.data_ptr(), s.data_ptr())


@pytest.mark.parametrize("given", [{}, {"ldb": 512}, {"b_scale_ld": 4}, {"ldb": 512, "b_scale_ld": 4}])
def test_group_strides_of_padded_weights(call, given):
    groups, n, k, m = 4, 5, 500, 130
    b, bs = bytes_(groups, 256, 512)[:, :m, :k], floats(groups, 3, 4)[:, :2]
    got = call(cm.MatmulKernelFp8Grouped, bytes_(n, k), floats(4, n), b, bs, zeros(n, m), zeros(groups + 1, dtype=torch.int32), groups, n, k, m, **given)
    assert (got.ldb, got.b_lds, got.b_gs, got.bs_gs) == (512, 4, 256 * 512, 12)


def test_strides_that_are_given_are_taken(call):
    x, q, s = zeros(3, 4, 128), bytes_(3, 4, 128), floats(3, 1, 4)
    got = call(cm.QuantKernelFp8, x, q, s, 2, 128, 3, ldx=256, x_batch_stride=512, q_batch_stride=300, ldq=128, scale_batch_stride=3)
    assert (got.ldx, got.x_bs, got.ldq, got.q_bs, got.lds, got.s_bs) == (256, 512, 128, 300, 4, 3)


def test_flat_and_two_dimensional_batches_are_dense(call):
    x, q, s = zeros(3 * 4, 128), bytes_(3 * 4 * 128), floats(3, 4)
    got = call(cm.QuantKernelFp8, x, q, s, 4, 128, 3)
    assert (got.ldx, got.x_bs, got.ldq, got.q_bs, got.lds, got.s_bs) == (128, 512, 128, 512, 4, 4)
    got = call(cm.QuantKernelFp8, 1 << 20, 1 << 21, 1 << 22, 4, 128, 3, ldx=130, x_type=cm.T_F16)
    assert (got.ldx, got.x_bs, got.q_bs, got.s_bs) == (130, 520, 512, 4)


def test_leading_dimensions_that_lie_evenly_are_one_batch(call):
    x, q, s = zeros(2, 3, 8, 128)[:, :, :4], bytes_(2, 3, 4, 128), floats(2, 3, 1, 4)
    got = call(cm.QuantKernelFp8, x, q, s, 4, 128, 6)
    assert (got.x_bs, got.q_bs, got.s_bs) == (8 * 128, 512, 4)
    got = call(cm.QuantKernelFp8, zeros(6, 8, 128)[:, :4].unsqueeze(1), q, s, 4, 128, 6)     # a dimension of one has no stride
    assert got.x_bs == 8 * 128
    got = call(cm.QuantKernelFp8, zeros(1, 4, 128).expand(6, 4, 128), q, s, 4, 128, 6)       # one x for all
    assert (got.ldx, got.x_bs) == (128, 0)
    with pytest.raises(ValueError):                                                          # a gap after three matrices
        call(cm.QuantKernelFp8, zeros(2, 4, 4, 128)[:, :3], q, s, 4, 128, 6)


@pytest.mark.parametrize("given", [{}, {"ldx": 128}])
def test_too_few_matrices_are_refused(call, given):
    with pytest.raises(ValueError):
        call(cm.QuantKernelFp8, zeros(3, 8, 128)[:2, :4], bytes_(3, 4, 128), floats(3, 1, 4), 4, 128, 3, **given)


# ---- a call stays inside the tensors that it is given ----------------------------------------------------
def quant(x, q, s, rows, cols, batch=1, **given):
    return cm.QuantKernelFp8, (x, q, s, rows, cols, batch), given


BEYOND = {   # views whose storage goes on behind them
    "batch of a matrix": quant(zeros(3 * 4, 128)[:4], bytes_(3, 4, 128), floats(3, 1, 4), 4, 128, 3),
    "output batch of a matrix": quant(zeros(3, 4, 128), bytes_(3 * 4, 128)[:8], floats(3, 1, 4), 4, 128, 3),
    "scales of a matrix": quant(zeros(3, 4, 128), bytes_(3, 4, 128), floats(3, 4)[:2], 4, 128, 3),
    "rows at a given pitch": quant(zeros(8, 128)[:4], bytes_(8, 128), floats(1, 8), 8, 128, ldx=128),
    "output rows at a given pitch": quant(zeros(8, 128), bytes_(8, 128)[:7], floats(1, 8), 8, 128, ldq=128),
    "a wider pitch than its own": quant(zeros(8, 256)[:, :128], bytes_(8, 128), floats(1, 8), 8, 128, ldx=257),
    "a given batch stride": quant(zeros(4, 4, 128)[:3], bytes_(3, 4, 128), floats(3, 1, 4), 4, 128, 3, x_batch_stride=600),
    "weights of the groups": (cm.MatmulKernelFp8Grouped, (bytes_(5, 128), floats(1, 5), bytes_(4 * 64, 128)[:64], floats(4, 1, 1), zeros(5, 64),
                                                         zeros(5, dtype=torch.int32), 4, 5, 128, 64), {}),
    "a number": (cm.MatmulKernelFp8, (bytes_(2, 128), floats(2)[0], bytes_(1, 128), floats(1), zeros(2, 1), 2, 128, 1), {}),
}


@pytest.mark.parametrize("which", BEYOND)
def test_nothing_beyond_a_tensor_is_reached(call, which):
    entry, args, given = BEYOND[which]
    with pytest.raises(ValueError):
        call(entry, *args, **given)


def test_all_of_a_tensor_may_be_reached(call):
    wide = zeros(8, 256)[:, :128]
    assert call(cm.QuantKernelFp8, wide, bytes_(8, 128), floats(1, 8), 8, 128, ldx=256).ldx == 256
    assert call(cm.QuantKernelFp8, wide, bytes_(8, 128), floats(4, 2), 2, 128, 4).x_bs == 512
    assert call(cm.QuantKernelFp8, zeros(4, 4, 128)[:3], bytes_(3, 4, 128), floats(3, 1, 4), 4, 128, 3, x_batch_stride=512).x_bs == 512
    assert call(cm.MatmulKernelFp8, bytes_(1, 128), floats(2)[0], bytes_(1, 128), floats(1), zeros(1, 1), 1, 128, 1).n == 1
    assert call(cm.QuantKernelFp8, zeros(0, 128), bytes_(0, 128), floats(1, 0), 0, 128).rows == 0
