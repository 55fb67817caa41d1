"""What the block-scaled 8-bit entries refuse, checked through the C ABI without a GPU: arguments are
looked at before the library is entered, so a refused call answers CM_EINVAL / CM_EUNSUPPORTED
before cm_init, and an allowed one CM_ENOINIT.  Addresses here are never dereferenced."""
import ctypes as C

import pytest

from cormorant_b200 import _lib

P = 1 << 20                       # an aligned address
EINVAL, EUNSUPPORTED, ENOINIT = _lib.CM_EINVAL, _lib.CM_EUNSUPPORTED, _lib.CM_ENOINIT


@pytest.fixture(scope="module")
def L():
    L = _lib.lib()
    if L.cm_device() >= 0:
        pytest.skip("already initialised in this process")
    return L


QUANT = dict(x=P, x_type=3, q=P, scale=P, rows=5, cols=300, batch=1, ldx=300, ldq=300, lds=5, x_bs=1500, q_bs=1500,
             s_bs=15, format=0, block_rows=1)
NORM = dict(x=P, resid=P, weight=P, resid_out=P, y=P, q=P, scale=P, rows=5, cols=300, ldx=300, ldr=300, ldo=300, ldy=300,
            ldq=300, lds=5, type=3, weight_type=1, eps=1e-6, format=0)
MATMUL = dict(a=P, a_scale=P, b=P, b_scale=P, c=P, n=5, k=300, m=200, lda=300, a_lds=5, ldb=300, b_lds=3, ldc=200,
              a_format=0, b_format=1, c_type=3)
GROUPED = dict(a=P, a_scale=P, b=P, b_scale=P, c=P, offsets=P, groups=4, n=5, k=300, m=200, lda=300, a_lds=5, ldb=300,
               b_lds=3, b_gs=60000, bs_gs=6, ldc=200, a_format=0, b_format=1, c_type=3)
CALLS = {"quant": ("cm_quant_fp8", QUANT), "norm": ("cm_rmsnorm_fp8", NORM), "matmul": ("cm_matmul_fp8", MATMUL),
         "grouped": ("cm_matmul_fp8_grouped", GROUPED)}


def call(L, which, **change):
    name, args = CALLS[which]
    assert set(change) <= set(args), set(change) - set(args)
    return getattr(L, name)(*{**args, **change}.values())


@pytest.mark.parametrize("which", CALLS)
def test_allowed_calls_reach_the_library(L, which):
    assert call(L, which) == ENOINIT
    name, args = CALLS[which]
    assert getattr(L, name + "_async")(*args.values(), None) == ENOINIT


ALLOWED = [
    ("quant", dict(rows=0)), ("quant", dict(cols=0, x=None)), ("quant", dict(batch=0)),
    ("quant", dict(rows=1, ldx=0, ldq=0)),                       # one row has no pitch
    ("quant", dict(block_rows=128, lds=3)),
    ("quant", dict(batch=3, x_bs=0)),                            # one x for all
    ("quant", dict(x=P + 2, q=P + 1, ldq=301)),                  # element alignment only
    ("norm", dict(resid=None, resid_out=None, weight=None)), ("norm", dict(y=None)), ("norm", dict(q=None, scale=None)),
    ("norm", dict(rows=0)), ("norm", dict(eps=0.0)), ("norm", dict(cols=32768, ldx=32768, ldr=32768, ldo=32768, ldy=32768, ldq=32768)),
    ("matmul", dict(n=0)), ("matmul", dict(k=0, a=None, b=None, a_scale=None, b_scale=None)), ("matmul", dict(m=0)),
    ("matmul", dict(a=P + 1, b=P + 3)), ("matmul", dict(c_type=0)),
    ("grouped", dict(groups=0)), ("grouped", dict(n=0)), ("grouped", dict(groups=1024)), ("grouped", dict(b_gs=0, bs_gs=0)),
]


@pytest.mark.parametrize("which,change", ALLOWED, ids=lambda v: v if isinstance(v, str) else "-".join(v))
def test_edges_that_are_allowed(L, which, change):
    assert call(L, which, **change) == ENOINIT, L.cm_last_error()


REFUSED = [
    ("quant", dict(x=None)), ("quant", dict(q=None)), ("quant", dict(scale=None)), ("quant", dict(x_type=4)),
    ("quant", dict(format=2)), ("quant", dict(block_rows=64)), ("quant", dict(ldx=299)), ("quant", dict(ldq=299)),
    ("quant", dict(lds=4)), ("quant", dict(block_rows=128, rows=129, lds=2)), ("quant", dict(x=P + 1)),
    ("quant", dict(x_type=1, x=P + 2)), ("quant", dict(scale=P + 2)), ("quant", dict(ldx=1 << 59)),
    ("quant", dict(ldq=1 << 63)), ("quant", dict(batch=2, q_bs=1499)), ("quant", dict(batch=2, s_bs=14)),
    ("quant", dict(batch=1 << 31, x_bs=1 << 40)),
    ("norm", dict(x=None)), ("norm", dict(y=None, q=None, scale=None)), ("norm", dict(q=None)), ("norm", dict(scale=None)),
    ("norm", dict(resid=None)), ("norm", dict(type=9)), ("norm", dict(weight_type=7)), ("norm", dict(format=3)),
    ("norm", dict(ldx=10)), ("norm", dict(ldr=10)), ("norm", dict(ldo=10)), ("norm", dict(ldy=10)), ("norm", dict(ldq=10)),
    ("norm", dict(lds=4)), ("norm", dict(eps=-1e-6)), ("norm", dict(eps=float("nan"))), ("norm", dict(eps=float("inf"))),
    ("norm", dict(resid=P + 1)), ("norm", dict(weight=P + 2)), ("norm", dict(ldx=1 << 60)),
    ("matmul", dict(a=None)), ("matmul", dict(b=None)), ("matmul", dict(a_scale=None)), ("matmul", dict(b_scale=None)),
    ("matmul", dict(c=None)), ("matmul", dict(a_format=2)), ("matmul", dict(b_format=9)), ("matmul", dict(c_type=5)),
    ("matmul", dict(lda=299)), ("matmul", dict(ldb=299)), ("matmul", dict(ldc=199)), ("matmul", dict(a_lds=4)),
    ("matmul", dict(b_lds=2)), ("matmul", dict(c=P + 1)), ("matmul", dict(a_scale=P + 2)), ("matmul", dict(b_scale=P + 1)),
    ("matmul", dict(lda=1 << 62)), ("matmul", dict(ldc=1 << 60)),
    ("grouped", dict(offsets=None)), ("grouped", dict(offsets=P + 2)), ("grouped", dict(b_gs=1 << 60)), ("grouped", dict(lda=299)),
    ("grouped", dict(c=None)),
]


@pytest.mark.parametrize("which,change", REFUSED, ids=lambda v: v if isinstance(v, str) else "-".join(v))
def test_bad_arguments_are_refused(L, which, change):
    assert call(L, which, **change) == EINVAL
    assert CALLS[which][0].encode() in L.cm_last_error()


# Outputs of batch steps may lie behind each other or, row by row, side by side; not in each other.
SIDE_BY_SIDE = [(dict(batch=2, q_bs=300, ldq=600), ENOINIT), (dict(batch=3, s_bs=5, lds=15), ENOINIT), (dict(batch=2, rows=1, q_bs=300, s_bs=1, lds=2), ENOINIT),
                (dict(batch=2, block_rows=128, rows=200, q_bs=300, ldq=700, s_bs=3, lds=6), ENOINIT), (dict(batch=2, q_bs=299, ldq=600), EINVAL),
                (dict(batch=2, q_bs=300, ldq=599), EINVAL), (dict(batch=3, s_bs=4, lds=15), EINVAL), (dict(batch=3, s_bs=5, lds=14), EINVAL),
                (dict(batch=2, q_bs=0, ldq=600), EINVAL), (dict(batch=2, cols=128, s_bs=4), EINVAL)]


@pytest.mark.parametrize("change,want", SIDE_BY_SIDE, ids=lambda v: "-".join(f"{k}{x}" for k, x in v.items()) if isinstance(v, dict) else str(v))
def test_outputs_of_batch_steps(L, change, want):
    assert call(L, "quant", **change) == want, L.cm_last_error()


@pytest.mark.parametrize("which,change", [
    ("norm", dict(type=0)), ("norm", dict(weight_type=0)),
    ("norm", dict(cols=32769, ldx=32769, ldr=32769, ldo=32769, ldy=32769, ldq=32769)),
    ("grouped", dict(groups=1025)), ("matmul", dict(n=1 << 31, a_lds=1 << 31)), ("matmul", dict(k=1 << 31, lda=1 << 31, ldb=1 << 31, b_lds=1 << 24)),
], ids=lambda v: v if isinstance(v, str) else "-".join(v))
def test_what_is_not_implemented_says_so(L, which, change):
    assert call(L, which, **change) == EUNSUPPORTED
    assert CALLS[which][0].encode() in L.cm_last_error()


def test_python_entries_refuse_host_tensors_and_wrong_types():
    import torch

    import cormorant_b200 as cm
    x, q, s = torch.zeros(4, 128), torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4)
    with pytest.raises(TypeError):
        cm.QuantKernelFp8(x, q, s, 4, 128)
    with pytest.raises(TypeError):                       # a raw address has no type of its own
        cm.QuantKernelFp8(P, P, P, 4, 128)
    with pytest.raises(TypeError):
        cm.MatmulKernelFp8(P, P, P, P, P, 4, 128, 128)
    assert C.sizeof(C.c_uint64) == 8
