"""Block-scaled 8-bit floating point on the GPU against plain implementations in 64 bits.

Tolerances are derived, with u = 2^-24 (half a step of fp32, relative) and h(T) = finfo(T).eps / 2:

quantisation  A, A / F and F / A are single fp32 operations on exact values, so scales equal the
              fp32 formula's and q equals its rounding; against 64 bits |q * scale - x| is at most
              half a step of the format (2^-4 or 2^-3 of |x|, or half the smallest subnormal times
              the scale) and the two fp32 roundings of x * (F / A) and one of the scale (4u |x|).
norm          h is one rounding (u); the squares' sum is of positive terms, at most 8 + 4 + 5 + 5
              roundings deep (22u); with the terms' own 3u, the division by the width, eps, root and
              reciprocal: 25u / 2 + 4u; times h and weight: 3u.  24u relative covers y before its
              own rounding.
product       the products of two 8-bit values are exact in fp32.  A block of 128 is summed by the
              tensor cores with an error of at most one step (2u) of the sum of magnitudes per
              addition: 256u; scaling and adding ceil(k/128) blocks (and up to eight partial sums of
              them) adds 2u a block and 8u:  |c - exact| <= (264 + 2 ceil(k/128)) u S + h(T) |c|
              with S = the same sum over magnitudes.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
HALF_STEP = {torch.float8_e4m3fn: 2.0 ** -4, torch.float8_e5m2: 2.0 ** -3}
HALF_SUBNORMAL = {torch.float8_e4m3fn: 2.0 ** -10, torch.float8_e5m2: 2.0 ** -17}
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
F32, F16, BF16, Q88 = torch.float32, torch.float16, torch.bfloat16, torch.int16
TINY = 2.0 ** -100


def up(v):
    return -(-v // 128)


def values(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    return x * (1 + 9 * (torch.rand(shape[-1], generator=g) < 0.05))


def typed(x, t):
    return (x * 256).round().clamp(-32768, 32767).to(Q88) if t == Q88 else x.to(t)


def real(x):
    return x.double() / 256 if x.dtype == Q88 else x.double()


def half(t):
    return torch.finfo(t).eps / 2


def expand(scale, rows, cols, block_rows):
    """Scales as stored -> one per element [rows][cols], in 64 bits."""
    s = scale.double().cpu()
    if block_rows == 1:
        return s.t().repeat_interleave(128, 1)[:rows, :cols]
    return s.repeat_interleave(128, 0).repeat_interleave(128, 1)[:rows, :cols]


def plain_quant(x, fmt, block_rows):
    """The fp32 formula on the CPU: (q as fp32 values, scale [row blocks][column blocks])."""
    rows, cols = x.shape
    p = torch.nn.functional.pad(x.float(), (0, -cols % 128, 0, -rows % block_rows))
    p = p.reshape(p.shape[0] // block_rows, block_rows, up(cols), 128)
    top = p.abs().amax(dim=(1, 3)).clamp_min(TINY)
    f = LARGEST[fmt]
    q = (p * (torch.tensor(f) / top)[:, None, :, None]).clamp(-f, f).to(fmt).float()
    return q.reshape(-1, up(cols) * 128)[:rows, :cols], top / f


def pitched(x, pitch, offset=0, poison=None):
    """x [rows][cols] on the GPU in rows `pitch` elements apart, starting `offset` elements into a buffer."""
    rows, cols = x.shape
    b = torch.zeros(offset + rows * pitch + 64, dtype=x.dtype if x.dtype not in LARGEST else torch.uint8, device="cuda")
    if poison is not None:
        b.fill_(poison)
    b = b if x.dtype not in LARGEST else b.view(x.dtype)
    v = b[offset: offset + rows * pitch].view(rows, pitch)[:, :cols]
    if x.dtype in LARGEST:
        v.view(torch.uint8).copy_(x.view(torch.uint8))
    else:
        v.copy_(x)
    return v


# ---- quantisation ---------------------------------------------------------------------------------
QUANT = [  # rows, cols, type, format, block_rows, x pitch, q pitch, element offset
    (1, 1, BF16, E4, 1, None, None, 0), (1, 128, F16, E4, 1, None, None, 0), (3, 127, F32, E5, 1, None, None, 0),
    (7, 129, BF16, E4, 1, 136, 136, 0), (8, 1000, F16, E5, 1, None, None, 0), (33, 1001, F32, E4, 1, None, None, 0),
    (65, 640, BF16, E4, 1, 656, 672, 8), (9, 512, BF16, E4, 1, None, 515, 1), (16, 4096, Q88, E4, 1, None, None, 0),
    (300, 515, Q88, E5, 1, None, None, 0), (2, 20000, BF16, E5, 1, None, None, 0),
    (1, 1, F32, E4, 128, None, None, 0), (128, 128, BF16, E4, 128, None, None, 0), (129, 257, F16, E5, 128, None, None, 0),
    (200, 384, F32, E4, 128, 388, 400, 4), (300, 1000, BF16, E4, 128, None, None, 0), (257, 129, Q88, E4, 128, None, None, 3),
]


@pytest.mark.parametrize("rows,cols,t,fmt,br,ldx,ldq,off", QUANT)
def test_quant(cm, rows, cols, t, fmt, br, ldx, ldq, off):
    x = typed(values(rows * 1009 + cols, rows, cols), t)
    x[0, : min(cols, 128)] = 0                                    # an empty block
    if rows > 2:
        x[2] = (x[2].float() * 2.0 ** -7).to(t)
    want_q, want_s = plain_quant(real(x).float(), fmt, br)
    ldx, ldq = ldx or cols, ldq or cols
    xd = pitched(x, ldx, off)
    q = pitched(torch.zeros(rows, cols, dtype=torch.uint8), ldq, off, poison=0xA5)
    shape = (up(cols), rows) if br == 1 else (up(rows), up(cols))
    scale = torch.full((shape[0] + 1, shape[1] + 3), -7.0, device="cuda")     # a pitch, and a row more
    cm.QuantKernelFp8(xd, q.view(fmt), scale, rows, cols, block_rows=br)
    got_s = scale[: shape[0], : shape[1]].cpu()
    assert torch.equal(got_s, want_s.t() if br == 1 else want_s)
    assert (scale[shape[0]] == -7).all() and (scale[:, shape[1]:] == -7).all()
    got = q.view(fmt).float().cpu()
    assert torch.equal(got, want_q)
    if ldq > cols and rows > 1:                                    # the gaps between rows are left alone
        gaps = q.as_strided((rows - 1, ldq - cols), (ldq, 1), q.storage_offset() + cols)
        assert (gaps == 0xA5).all()
    s = expand(got_s, rows, cols, br)
    err = (got.double() * s - real(x)).abs()
    assert (err <= torch.maximum(HALF_STEP[fmt] * real(x).abs(), HALF_SUBNORMAL[fmt] * s) + 4 * U * real(x).abs()).all()


@pytest.mark.parametrize("br", [1, 128])
def test_quant_batch_and_broadcast(cm, br):
    batch, rows, cols = 3, 130, 200
    x = values(5, batch, rows, cols).to(BF16).cuda()
    q = torch.empty(batch, rows, cols, dtype=E4, device="cuda")
    shape = (up(cols), rows) if br == 1 else (up(rows), up(cols))
    scale = torch.empty(batch, *shape, device="cuda")
    cm.QuantKernelFp8(x, q, scale, rows, cols, batch, block_rows=br)
    for z in range(batch):
        want_q, want_s = plain_quant(x[z].float().cpu(), E4, br)
        assert torch.equal(q[z].float().cpu(), want_q)
        assert torch.equal(scale[z].cpu(), want_s.t() if br == 1 else want_s)
    cm.QuantKernelFp8(x, q, scale, rows, cols, batch, x_batch_stride=0, block_rows=br)
    assert torch.equal(q[2].view(torch.uint8), q[0].view(torch.uint8)) and torch.equal(scale[2], scale[0])


@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("batch,rows,cols", [(3, 130, 200), (4, 1, 300), (2, 70, 1024)])
def test_quant_batch_side_by_side(cm, br, batch, rows, cols):
    """Batch steps whose output rows lie between each other's: one operand of all steps' columns, scales of all steps' rows."""
    x = values(8, batch, rows, cols).to(BF16).cuda()
    q = torch.full((rows, batch, cols), 0x55, dtype=torch.uint8, device="cuda").view(E4)
    outer, inner = (up(cols), rows) if br == 1 else (up(rows), up(cols))
    scale = torch.full((outer, batch, inner), -7.0, device="cuda")
    cm.QuantKernelFp8(x, q.permute(1, 0, 2), scale.permute(1, 0, 2), rows, cols, batch, block_rows=br)
    for z in range(batch):
        want_q, want_s = plain_quant(x[z].float().cpu(), E4, br)
        assert torch.equal(q[:, z].float().cpu(), want_q)
        assert torch.equal(scale[:, z].cpu(), want_s.t() if br == 1 else want_s)


@pytest.mark.parametrize("fmt", [E4, E5])
@pytest.mark.parametrize("br", [1, 128])
def test_quant_infinities_nan_and_extremes(cm, fmt, br):
    rows, cols = 128, 640
    x = values(6, rows, cols)
    x[1, 5], x[2, 130], x[3, 300] = float("inf"), float("nan"), -float("inf")
    x[:, 384:512] *= 2.0 ** -120
    x[:, 512:] = x[:, 512:].sign() * torch.finfo(F32).max
    q = torch.empty(rows, cols, dtype=fmt, device="cuda")
    scale = torch.empty(up(cols) if br == 1 else 1, rows if br == 1 else up(cols), device="cuda")
    cm.QuantKernelFp8(x.cuda(), q, scale, rows, cols, block_rows=br)
    got, s = q.float().cpu(), expand(scale, rows, cols, br)
    inf_rows, nan_rows = ([1], [2]) if br == 1 else (range(rows), range(rows))
    for r in inf_rows:
        b = slice(0, 128)
        assert torch.isinf(s[r, b]).all()
        assert torch.equal(torch.isnan(got[r, b]), torch.isinf(x[r, b])) and (got[r, b][torch.isfinite(x[r, b])] == 0).all()
    for r in nan_rows:
        assert torch.isnan(s[r, 128:256]).all() and torch.isnan(got[r, 128:256]).all()
    assert torch.isfinite(got[:, 384:]).all() and torch.isfinite(s[:, 384:]).all()
    if br == 1:
        keep = [r for r in range(rows) if r not in (1, 2, 3)]
        want_q, _ = plain_quant(x[keep], fmt, 1)
        assert torch.equal(got[keep], want_q)


# ---- norm -------------------------------------------------------------------------------------------
NORM = [  # rows, cols, type, weight type, format, resid, resid_out, y, q, pitch, element offset
    (1, 1, F32, F32, E4, 1, 1, 1, 1, None, 0), (1, 4096, BF16, BF16, E4, 1, 1, 0, 1, None, 0), (5, 127, F16, F32, E5, 1, 0, 1, 1, None, 0),
    (3, 128, BF16, None, E4, 0, 0, 1, 0, None, 0), (9, 1001, F32, F32, E4, 0, 0, 1, 1, None, 0), (70, 1024, F16, F16, E5, 1, 1, 1, 1, None, 0),
    (4, 1025, BF16, F32, E4, 1, 1, 1, 1, 1032, 0), (700, 513, BF16, BF16, E4, 1, 1, 1, 1, None, 0), (6, 5000, BF16, BF16, E4, 1, 1, 1, 1, 5008, 8),
    (601, 4096, F16, F16, E4, 1, 1, 0, 1, None, 0), (650, 4104, BF16, F32, E4, 1, 1, 1, 1, None, 0), (2, 20000, BF16, BF16, E5, 1, 1, 1, 1, None, 0),
    (3, 32768, F32, F32, E4, 1, 1, 1, 1, None, 0), (2, 32767, F16, F16, E4, 0, 0, 1, 1, None, 0), (600, 16384, BF16, BF16, E4, 0, 0, 0, 1, None, 0),
    (640, 264, F32, F32, E4, 1, 1, 1, 1, None, 1), (2000, 200, BF16, BF16, E4, 1, 1, 1, 1, None, 0), (1, 300, F32, F32, E4, 0, 0, 0, 1, None, 0),
    (700, 8192, BF16, BF16, E4, 1, 1, 0, 1, None, 0),
]


@pytest.mark.parametrize("rows,cols,t,wt,fmt,with_r,with_o,with_y,with_q,pitch,off", NORM)
def test_rmsnorm(cm, rows, cols, t, wt, fmt, with_r, with_o, with_y, with_q, pitch, off):
    eps = 1e-5
    x, r = values(rows + cols, rows, cols).to(t), values(rows + cols + 1, rows, cols, scale=3.0).to(t)
    x[0], r[0] = 0, 0                                              # mean square 0: y = 0 * 1 / sqrt(eps)
    w = None if wt is None else (1 + 0.2 * values(cols, cols)).to(wt)
    h = x.double() + (r.double() if with_r else 0)
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * (1 if w is None else w.double())
    ld = pitch or cols
    out = lambda on: pitched(torch.zeros(rows, cols, dtype=t), ld, off, poison=-3.0) if on else None  # noqa: E731
    ro, yo = out(with_o), out(with_y)
    q = pitched(torch.zeros(rows, cols, dtype=torch.uint8), ld, off, poison=0xA5) if with_q else None
    scale = torch.full((up(cols), rows), -7.0, device="cuda") if with_q else None
    cm.RmsNormKernelFp8(pitched(x, ld, off), None if w is None else w.cuda(), q.view(fmt) if with_q else None, scale, rows, cols,
                        eps=eps, resid=pitched(r, ld, off) if with_r else None, resid_out=ro, y=yo)
    if with_o:
        assert ((ro.double().cpu() - h).abs() <= (half(t) + 2 * U) * h.abs() + 2.0 ** -25).all()
    tol = 24 * U * y.abs()
    if with_y:     # 2^-25: half the smallest fp16 subnormal
        assert ((yo.double().cpu() - y).abs() <= tol + half(t) * y.abs() + 2.0 ** -25).all()
    if with_q:
        p = torch.nn.functional.pad(y.abs(), (0, -cols % 128)).reshape(rows, up(cols), 128).amax(2).clamp_min(TINY)
        want_s = (p / LARGEST[fmt]).t()
        assert ((scale.double().cpu() - want_s).abs() <= 25 * U * want_s).all()
        s = expand(scale, rows, cols, 1)
        err = (q.view(fmt).double().cpu() * s - y).abs()
        assert (err <= torch.maximum(HALF_STEP[fmt] * y.abs(), HALF_SUBNORMAL[fmt] * s) + 32 * U * y.abs()).all()
    if ld > cols and rows > 1:
        for o, v in ((ro, -3.0), (yo, -3.0), (q, 0xA5)):
            if o is not None:
                assert (o.as_strided((rows - 1, ld - cols), (ld, 1), o.storage_offset() + cols) == v).all()


# Squares that leave fp32: rows of one block, of a part of a warp, of several warps, and of the widest CTA, each with
# ordinary rows beside the ones whose squares overflow or vanish.
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(9, 1), (70, 100), (41, 777), (13, 1024), (700, 2056), (5, 20000)])
@pytest.mark.parametrize("eps", [0.0, 1e-5, 2.0 ** -130])
def test_rmsnorm_large_and_small_rows(cm, t, rows, cols, eps):
    x, w = values(rows, rows, cols), (1 + 0.2 * values(cols, cols)).to(t)
    x[x == 0] = 1.0
    exponents = torch.tensor([0, 62, -70, 100, -110, 123, -125, 64, -40])[torch.arange(rows) % 9]
    x = (x.clamp(-8, 8).double() * (2.0 ** exponents.double())[:, None]).to(t)
    r = torch.zeros_like(x)
    ro, y = torch.empty(rows, cols, dtype=t, device="cuda"), torch.empty(rows, cols, dtype=t, device="cuda")
    q, s = torch.empty(rows, cols, dtype=E4, device="cuda"), torch.empty(up(cols), rows, device="cuda")
    cm.RmsNormKernelFp8(x.cuda(), w.cuda(), q, s, rows, cols, eps=eps, resid=r.cuda(), resid_out=ro, y=y)
    assert torch.equal(ro.cpu(), x)
    h = x.double()
    want = h / torch.sqrt((h * h).mean(1, keepdim=True) + float(torch.tensor(eps))) * w.double()
    # 24u and the output's rounding as above; results below 2^-126 (rows far below eps) are multiples of 2^-149, three roundings
    err = (y.double().cpu() - want).abs()
    assert (err <= (24 * U + half(t)) * want.abs() + (3 * 2.0 ** -150 if t == F32 else 2.0 ** -134 + 2 * 2.0 ** -150)).all()
    sc = expand(s, rows, cols, 1)
    err = (q.double().cpu() * sc - want).abs()
    assert (err <= torch.maximum(HALF_STEP[E4] * want.abs(), HALF_SUBNORMAL[E4] * sc) + 32 * U * want.abs() + 4 * 2.0 ** -150).all()


@pytest.mark.parametrize("rows,cols", [(5, 4096), (700, 1000)])
def test_rmsnorm_in_place(cm, rows, cols):
    x, r, w = values(1, rows, cols).to(BF16).cuda(), values(2, rows, cols).to(BF16).cuda(), values(3, cols).to(BF16).cuda()
    q1, q2 = (torch.empty(rows, cols, dtype=E4, device="cuda") for _ in range(2))
    s1, s2 = (torch.empty(up(cols), rows, device="cuda") for _ in range(2))
    ro, y = torch.empty_like(x), torch.empty_like(x)
    cm.RmsNormKernelFp8(x, w, q1, s1, rows, cols, resid=r, resid_out=ro, y=y)
    cm.RmsNormKernelFp8(x, w, q2, s2, rows, cols, resid=r, resid_out=r, y=x)       # over the inputs
    assert torch.equal(r, ro) and torch.equal(x, y) and torch.equal(s1, s2)
    assert torch.equal(q1.view(torch.uint8), q2.view(torch.uint8))


def test_rmsnorm_nan_stays_in_its_row(cm):
    rows, cols = 6, 640
    x = values(4, rows, cols)
    x[1, 7], x[4, 630] = float("nan"), float("inf")
    y = torch.empty(rows, cols, device="cuda")
    q, s = torch.empty(rows, cols, dtype=E4, device="cuda"), torch.empty(up(cols), rows, device="cuda")
    cm.RmsNormKernelFp8(x.cuda(), None, q, s, rows, cols, y=y)
    bad = torch.tensor([False, True, False, False, True, False])
    assert torch.equal(~torch.isfinite(y.cpu()).all(1), bad)
    assert torch.equal(~torch.isfinite(s.cpu()).all(0), bad)
    assert torch.isfinite(q.float().cpu()[~bad]).all()


def ring(rows, cols, t, pitch, offset):
    """A byte buffer of 0xA5 and the view of [rows][cols] elements of t inside it."""
    size = t.itemsize
    b = torch.full(((offset + rows * pitch + 64) * size,), 0xA5, dtype=torch.uint8, device="cuda")
    return b, b.view(t)[offset: offset + rows * pitch].view(rows, pitch)[:, :cols]


# The layout of the rows changes neither the formula nor the order of a sum: every offset gives the
# bits of the aligned call (which the tests above hold to 64 bits), and writes nothing beside its rows.
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("cols", [1, 7, 8, 9, 100, 127, 128, 130, 257, 384, 500, 1001, 1023, 1100])
def test_rows_at_every_offset(cm, t, cols):
    rows = 37
    aligned = -(-cols // 16) * 16
    x, r = pitched(values(cols, rows, cols).to(t), aligned), pitched(values(cols + 1, rows, cols).to(t), aligned)
    w = (1 + 0.2 * values(cols, cols)).to(t).cuda()
    make = lambda: [ring(rows, cols, d, aligned, 0)[1] for d in (t, t, torch.uint8, torch.uint8)] + [torch.empty(up(cols), rows, device="cuda") for _ in "12"]  # noqa: E731
    want = make()
    cm.RmsNormKernelFp8(x, w, want[2].view(E4), want[4], rows, cols, resid=r, resid_out=want[0], y=want[1])
    cm.QuantKernelFp8(x, want[3].view(E5), want[5], rows, cols)
    for i, off in enumerate([0, 1, 2, 3, 4, 5, 7, 8, 11, 15]):
        pitch = cols + (0, 1, 3, 8)[i % 4]
        xs, rs, ws = ring(rows, cols, t, pitch, off)[1].copy_(x), ring(rows, cols, t, pitch, (off * 3) % 8)[1].copy_(r), ring(1, cols, t, cols, off)[1][0].copy_(w)
        bufs = [ring(rows, cols, d, pitch, (off * k) % 16) for d, k in ((t, 1), (t, 5), (torch.uint8, 1), (torch.uint8, 3))]
        s1, s2 = torch.empty(up(cols), rows, device="cuda"), torch.empty(up(cols), rows, device="cuda")
        cm.RmsNormKernelFp8(xs, ws, bufs[2][1].view(E4), s1, rows, cols, resid=rs, resid_out=bufs[0][1], y=bufs[1][1])
        cm.QuantKernelFp8(xs, bufs[3][1].view(E5), s2, rows, cols)
        assert torch.equal(s1, want[4]) and torch.equal(s2, want[5]), off
        for (b, v), u in zip(bufs, want):
            assert torch.equal(v.contiguous().view(torch.uint8), u.contiguous().view(torch.uint8)), off
            v.view(torch.uint8).fill_(0xA5)
            assert (b == 0xA5).all(), off


@pytest.mark.parametrize("cols", [2 ** 32 - 1, 2 ** 32 - 8])
def test_quant_longest_row(cm, cols):
    """The columns of a 32-bit size's end, at odd addresses: offsets past 32 bits, no index that wraps."""
    tail = 1000 + cols % 128
    x = torch.zeros(cols, dtype=BF16, device="cuda")
    x[-tail:] = values(5, tail).to(BF16).cuda()
    x[:256] = values(6, 256).to(BF16).cuda()
    b = torch.full((cols + 8,), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.empty(up(cols), 1, device="cuda")
    for off in (1, 2, 3):
        q = b[off: off + cols]
        cm.QuantKernelFp8(x, q, s, 1, cols, fmt=0)
        first = (cols - tail) // 128 * 128
        for lo, hi in ((0, 256), (first, cols)):
            want_q, want_s = plain_quant(x[lo:hi].float().cpu()[None], E4, 1)
            assert torch.equal(q[lo:hi].view(E4).float().cpu()[None], want_q), off
            assert torch.equal(s[lo // 128: up(hi), 0].cpu(), want_s[0]), off
        assert (b[:off] == 0xA5).all() and (b[off + cols:] == 0xA5).all()
        b[-16:] = 0xA5
        b[:16] = 0xA5


@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("cols", [2 ** 32 - 1, 2 ** 32 - 5, 2 ** 32 - 127])
@pytest.mark.parametrize("behind", [float("nan"), 2.0 ** 100])
def test_quant_longest_row_takes_nothing_from_behind_it(cm, cols, br, behind):
    """The last block of a row that ends within 128 columns of 2^32: what follows the row in its last words stays out."""
    tail = 1000 + cols % 128
    b = torch.zeros(cols + 8, dtype=BF16, device="cuda")
    x = b[:cols]
    x[-tail:] = values(7, tail).to(BF16).cuda()
    b[cols:] = behind
    q, s = torch.empty(cols, dtype=E4, device="cuda"), torch.full((up(cols), 1) if br == 1 else (1, up(cols)), -7.0, device="cuda")
    cm.QuantKernelFp8(x, q, s, 1, cols, block_rows=br)
    first = (cols - tail) // 128 * 128
    want_q, want_s = plain_quant(x[first:].float().cpu()[None], E4, br)
    assert torch.equal(s.flatten()[first // 128:].cpu(), want_s.flatten())
    assert torch.equal(q[first:].float().cpu()[None], want_q)


@pytest.mark.parametrize("rows,cols", [(3000, 1), (5000, 120), (2500, 250), (1300, 640), (1200, 1500), (300, 9000)])
def test_rmsnorm_more_rows_than_a_pass(cm, rows, cols):
    x, w = values(rows, rows, cols).to(BF16), (1 + 0.2 * values(cols, cols)).to(BF16)
    y = torch.empty(rows, cols, dtype=BF16, device="cuda")
    q, s = torch.empty(rows, cols, dtype=E4, device="cuda"), torch.empty(up(cols), rows, device="cuda")
    cm.RmsNormKernelFp8(x.cuda(), w.cuda(), q, s, rows, cols, eps=1e-6, y=y)
    h = x.double()
    want = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * w.double()
    assert ((y.double().cpu() - want).abs() <= (24 * U + half(BF16)) * want.abs()).all()
    sc = expand(s, rows, cols, 1)
    err = (q.double().cpu() * sc - want).abs()
    assert (err <= torch.maximum(HALF_STEP[E4] * want.abs(), HALF_SUBNORMAL[E4] * sc) + 32 * U * want.abs()).all()


def test_rmsnorm_in_place_unaligned(cm):
    rows, cols = 700, 1001
    x, r, w = values(1, rows, cols).to(F16).cuda(), values(2, rows, cols).to(F16).cuda(), values(3, cols).to(F16).cuda()
    q1, q2 = (torch.empty(rows, cols, dtype=E5, device="cuda") for _ in range(2))
    s1, s2 = (torch.empty(up(cols), rows, device="cuda") for _ in range(2))
    ro, y = torch.empty_like(x), torch.empty_like(x)
    cm.RmsNormKernelFp8(x, w, q1, s1, rows, cols, resid=r, resid_out=ro, y=y)
    cm.RmsNormKernelFp8(x, w, q2, s2, rows, cols, resid=r, resid_out=r, y=x)
    assert torch.equal(r, ro) and torch.equal(x, y) and torch.equal(s1, s2)
    assert torch.equal(q1.view(torch.uint8), q2.view(torch.uint8))


# ---- products ---------------------------------------------------------------------------------------
def operands(seed, n, k, m, af=E4, bf=E4, groups=0):
    """(a, a_scale, b, b_scale) on the CPU: 8-bit values and scales as the quantising entries store them."""
    a, sa = plain_quant(values(seed, n, k), af, 1)
    shape = (groups,) if groups else ()
    w = torch.randn(*shape, m, k, generator=torch.Generator().manual_seed(seed + 1)) * 0.05
    if groups:
        both = [plain_quant(w[g], bf, 128) for g in range(groups)]
        b, sb = torch.stack([v[0] for v in both]), torch.stack([v[1] for v in both])
    else:
        b, sb = plain_quant(w, bf, 128)
    return a.to(af), sa.t().contiguous(), b.to(bf), sb


def product64(a, sa, b, sb):
    """The exact product and the same sum over magnitudes."""
    n, k = a.shape
    A = a.double() * expand(sa, n, k, 1)
    B = b.double() * expand(sb, b.shape[0], k, 128)
    return A @ B.t(), A.abs() @ B.abs().t()


def check_product(got, want, mag, k, t):
    tol = (264 + 2 * up(k)) * U * mag
    if t == Q88:          # floor to 1/256 and saturation: whole words, one off where the exact value is within tol of a border
        w = want * 256
        lo, hi = torch.floor(w - 256 * tol).clamp(-32768, 32767), torch.floor(w + 256 * tol).clamp(-32768, 32767)
        g = got.double()
        assert ((g >= lo) & (g <= hi)).all()
        return
    err = (got.double() - want).abs()
    bad = err > tol + half(t) * want.abs() + (2.0 ** -25 if t == F16 else 0)
    assert not bad.any(), (int(bad.sum()), float((err / (tol + 1e-300)).max()), bad.nonzero()[:4].tolist())


MATMUL = [  # n, k, m, c type, a format, b format
    (1, 1, 1, F32, E4, E4), (1, 16, 8, F32, E4, E4), (1, 128, 128, F32, E4, E4), (1, 4096, 256, BF16, E4, E4), (2, 100, 127, F32, E4, E5),
    (3, 129, 129, F16, E5, E4), (15, 1000, 130, F32, E5, E5), (16, 256, 128, BF16, E4, E4), (17, 1024, 513, F32, E4, E4),
    (31, 2049, 100, F32, E4, E4), (33, 513, 640, BF16, E4, E4), (64, 7168, 256, F32, E4, E4), (65, 640, 300, F16, E4, E4),
    (127, 384, 129, Q88, E4, E4), (128, 128, 128, F32, E4, E4), (129, 1000, 257, F32, E4, E5), (200, 515, 1001, BF16, E5, E4),
    (255, 256, 512, F32, E4, E4), (257, 129, 300, F32, E4, E4), (300, 1000, 1001, F32, E5, E4), (513, 2048, 640, F16, E4, E4),
    (1000, 512, 384, Q88, E4, E4), (1100, 1152, 1300, BF16, E4, E4), (4, 16384, 136, F32, E4, E4), (2048, 640, 16, F32, E4, E4),
    (777, 96, 2048, BF16, E4, E4),
    # K split over two, four and eight CTAs; tiles of 64, 128 and 256 tokens, several of a CTA
    (308, 2716, 129, F32, E4, E4), (163, 1794, 141, BF16, E4, E5), (1, 1545, 16, F32, E5, E4), (2413, 300, 135, F32, E4, E4),
    (1000, 700, 2049, F16, E4, E4), (3454, 100, 265, BF16, E4, E5), (520, 300, 1500, F32, E4, E4), (2720, 300, 797, F32, E5, E4),
    (1300, 1500, 2500, BF16, E4, E4), (1300, 1500, 2501, F32, E4, E4), (4000, 129, 1100, Q88, E4, E4), (1025, 515, 2100, F16, E4, E4),
]


@pytest.mark.parametrize("n,k,m,t,af,bf", MATMUL)
def test_matmul(cm, n, k, m, t, af, bf):
    a, sa, b, sb = operands(n + k + m, n, k, m, af, bf)
    want, mag = product64(a, sa, b, sb)
    c = torch.full((n + 1, m + 5), -3, dtype=t, device="cuda")
    cm.MatmulKernelFp8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, n, k, m)
    check_product(c[:n, :m].cpu(), want, mag, k, t)
    assert (c[n] == -3).all() and (c[:, m:] == -3).all()
    k16 = (k + 15) // 16 * 16                                      # the same operands in aligned rows: the same bits
    c2 = torch.full_like(c, -3)
    cm.MatmulKernelFp8(pitched(a, k16 + 16), sa.cuda(), pitched(b, k16 + 32), sb.cuda(), c2, n, k, m)
    assert torch.equal(c, c2)


# 256 x 128 tiles on pairs of SMs: one tile a pair and several, 1 to 9 blocks of K through four
# accumulators, an odd and an even number of weight blocks, every output type
PAIRS = [(300, 1000, 4001, BF16, E5, E4), (513, 300, 2100, F16, E4, E4), (700, 520, 1990, Q88, E4, E5), (4043, 69, 1162, F32, E4, E4),
         (3697, 143, 1717, BF16, E4, E4), (5000, 384, 900, F32, E4, E5), (3257, 543, 1987, F16, E5, E4), (4028, 836, 1040, F32, E4, E4)]


@pytest.mark.parametrize("n,k,m,t,af,bf", PAIRS)
def test_matmul_pairs(cm, n, k, m, t, af, bf):
    test_matmul(cm, n, k, m, t, af, bf)


PAIRS_GROUPED = [([700, 0, 1300, 2254], 3, 0, 190, 988, F32, E4, E4), ([1000, 1, 256, 1058], 0, 4, 307, 2234, BF16, E4, E5),
                 ([500, 700, 0, 300, 3, 335], 0, 0, 1096, 1890, F16, E4, E4)]


@pytest.mark.parametrize("sizes,before,behind,k,m,t,af,bf", PAIRS_GROUPED)
def test_grouped_pairs(cm, sizes, before, behind, k, m, t, af, bf):
    test_grouped(cm, sizes, before, behind, k, m, t, af, bf)


@pytest.mark.parametrize("n,k,m,off_a,off_b,off_c", [(5, 256, 130, 1, 0, 1), (130, 300, 200, 0, 3, 1), (300, 512, 256, 8, 8, 3)])
def test_matmul_unaligned_bases(cm, n, k, m, off_a, off_b, off_c):
    a, sa, b, sb = operands(n, n, k, m)
    want, mag = product64(a, sa, b, sb)
    c = pitched(torch.zeros(n, m, dtype=BF16), m + 1, off_c, poison=-3.0)
    wide = torch.zeros(up(k), n + 7, device="cuda")
    wide[:, 3: 3 + n] = sa.cuda()
    cm.MatmulKernelFp8(pitched(a, k, off_a), wide[:, 3: 3 + n], pitched(b, k, off_b), sb.cuda(), c, n, k, m)
    check_product(c.cpu(), want, mag, k, BF16)


def test_matmul_empty_sum_and_empty_sizes(cm):
    c = torch.full((5, 300), 7.0, device="cuda")
    cm.MatmulKernelFp8(0, 0, 0, 0, c, 5, 0, 300, a_scale_ld=5, b_scale_ld=0)
    assert (c == 0).all()
    c.fill_(7.0)
    a = torch.zeros(0, 128, dtype=E4, device="cuda")
    cm.MatmulKernelFp8(a, torch.zeros(1, 0, device="cuda"), torch.zeros(300, 128, dtype=E4, device="cuda"), torch.zeros(3, 1, device="cuda"), c, 0, 128, 300)
    assert (c == 7).all()


@pytest.mark.parametrize("n", [3, 40, 300])
def test_matmul_nan_and_infinity_stay_in_their_row_and_column(cm, n):
    k, m = 640, 300
    a, sa, b, sb = operands(9, n, k, m)
    want, mag = product64(a, sa, b, sb)
    ai = a.view(torch.uint8).clone()
    ai[1, 130] = 0x7F                                              # NaN in e4m3
    sa = sa.clone()
    sa[3, 2] = float("inf")                                        # a row whose block held an infinity
    bi = b.view(torch.uint8).clone()
    bi[200, 5] = 0xFF
    c = torch.empty(n, m, device="cuda")
    cm.MatmulKernelFp8(ai.view(E4).cuda(), sa.cuda(), bi.view(E4).cuda(), sb.cuda(), c, n, k, m)
    got = c.cpu()
    rows, cols = torch.arange(n), torch.arange(m)
    clean = ((rows != 1) & (rows != 2))[:, None] & (cols != 200)[None, :]
    assert not torch.isfinite(got[1]).any() and not torch.isfinite(got[2]).any() and torch.isnan(got[:, 200]).all()
    err = (got.double() - want).abs()
    assert (err <= (264 + 2 * up(k)) * U * mag + half(F32) * want.abs())[clean].all()


@pytest.mark.parametrize("n", [3, 40, 300, 1300])
@pytest.mark.parametrize("af,bf", [(E4, E4), (E5, E4), (E5, E5)])
@pytest.mark.parametrize("exponent", [-125, -127, -140, -149, -170])
def test_matmul_small_scales(cm, n, af, bf, exponent):
    """Scales whose products are just normal, subnormal and zero in fp32.  A scale of 2^-126 or more is one rounding (u,
    counted above), one below is off by 2^-150 at most, which the block's sum multiplies; results and their kb additions
    are multiples of 2^-149, off by half of it each."""
    k, m = 300, 1500 if n > 1000 else 130
    a, sa, b, sb = operands(n + 1, n, k, m, af, bf)
    sa, sb = (1 + 0.4 * torch.rand(sa.shape, generator=torch.Generator().manual_seed(1))) * 2.0 ** -64, \
             (1 + 0.4 * torch.rand(sb.shape, generator=torch.Generator().manual_seed(2))) * 2.0 ** (exponent + 64)
    want, mag = product64(a, sa, b, sb)
    lost = a.double().abs() @ b.double().abs().t() * 2.0 ** -150 if exponent < -126 else 0
    c = torch.empty(n, m, device="cuda")
    cm.MatmulKernelFp8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, n, k, m)
    err = (c.double().cpu() - want).abs()
    assert (err <= (264 + 2 * up(k)) * U * mag + half(F32) * want.abs() + lost + (up(k) + 9) * 2.0 ** -150).all()


def test_matmul_pitch_past_32_bits(cm):
    """Rows of a and c that lie more than 2^32 bytes apart."""
    n, k, m = 3, 256, 136
    a, sa, b, sb = operands(11, n, k, m)
    want, mag = product64(a, sa, b, sb)
    lda, ldc = (1 << 32) // 2 + 16, (1 << 32) // 4 + 8
    abuf = torch.zeros(2 * lda + k, dtype=torch.uint8, device="cuda")
    cbuf = torch.zeros(2 * ldc + m, dtype=F32, device="cuda")
    av, cv = abuf.as_strided((n, k), (lda, 1)).view(E4), cbuf.as_strided((n, m), (ldc, 1))
    av.view(torch.uint8).copy_(a.view(torch.uint8))
    cm.MatmulKernelFp8(av, sa.cuda(), b.cuda(), sb.cuda(), cv, n, k, m)
    check_product(cv.cpu(), want, mag, k, F32)
    q, s = torch.empty(n, m, dtype=E4, device="cuda"), torch.empty(up(m), n, device="cuda")
    cm.QuantKernelFp8(cv, q, s, n, m)
    want_q, _ = plain_quant(cv.cpu(), E4, 1)
    assert torch.equal(q.float().cpu(), want_q)


# ---- grouped ----------------------------------------------------------------------------------------
GROUPED = [  # row counts, rows before the first, rows behind the last, k, m, c type, formats
    ([5], 0, 0, 128, 128, F32, E4, E4), ([1, 1, 1, 1], 0, 0, 256, 136, BF16, E4, E4), ([0, 0, 3], 0, 2, 300, 100, F32, E4, E4),
    ([0, 0, 0], 2, 3, 256, 64, F32, E4, E4), ([17, 0, 1, 40], 3, 5, 515, 200, F16, E5, E4), ([129, 128, 127], 0, 1, 640, 260, F32, E4, E5),
    ([300, 0, 5, 211], 1, 0, 1000, 520, F32, E4, E4), ([2] * 40, 0, 0, 512, 128, BF16, E4, E4), ([600, 700], 0, 9, 256, 384, BF16, E4, E4),
    ([0, 513], 0, 0, 129, 130, Q88, E4, E4), ([1] * 100 + [0] * 900 + [30], 0, 0, 128, 32, F32, E4, E4), ([900, 20, 0, 400, 256, 100], 7, 13, 1152, 640, BF16, E4, E4),
    # as above: split K, wider tiles, several tiles of a CTA
    ([100, 0, 180], 0, 0, 1795, 17, F32, E4, E4), ([3, 550, 8], 1, 1, 2751, 20, F32, E4, E4), ([2] * 40, 0, 0, 512, 1024, BF16, E4, E4),
    ([1000, 0, 1395], 0, 5, 130, 140, F32, E4, E4), ([600, 1, 0, 1500, 700, 370], 2, 0, 200, 267, F16, E4, E5),
    ([900, 0, 1300, 213], 3, 4, 300, 914, F32, E4, E4), ([257, 0, 255, 900, 1], 0, 87, 600, 1300, BF16, E4, E4),
]


def grouped_want(a, sa, b, sb, ends, fill):
    n, m = a.shape[0], b.shape[1]
    want, mag = torch.full((n, m), fill, dtype=torch.float64), torch.zeros(n, m, dtype=torch.float64)
    for g, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if hi > lo:
            want[lo:hi], mag[lo:hi] = product64(a[lo:hi], sa[:, lo:hi], b[g], sb[g])
    return want, mag


@pytest.mark.parametrize("sizes,before,behind,k,m,t,af,bf", GROUPED)
def test_grouped(cm, sizes, before, behind, k, m, t, af, bf):
    ends = [before]
    for v in sizes:
        ends.append(ends[-1] + v)
    n = ends[-1] + behind
    a, sa, b, sb = operands(k + m, n, k, m, af, bf, groups=len(sizes))
    want, mag = grouped_want(a, sa, b, sb, ends, 0.0)
    c = torch.full((n, m), -3, dtype=t, device="cuda")
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    args = (off, len(sizes), n, k, m)
    cm.MatmulKernelFp8Grouped(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, *args)
    assert (c[: ends[0]] == -3).all() and (c[ends[-1]:] == -3).all()
    if ends[-1] > ends[0]:
        check_product(c[ends[0]: ends[-1]].cpu(), want[ends[0]: ends[-1]], mag[ends[0]: ends[-1]], k, t)
    k16 = (k + 15) // 16 * 16
    bp = torch.zeros(len(sizes), m, k16, dtype=torch.uint8, device="cuda").view(bf)
    bp[:, :, :k].view(torch.uint8).copy_(b.view(torch.uint8))
    c2 = torch.full_like(c, -3)
    cm.MatmulKernelFp8Grouped(pitched(a, k16), sa.cuda(), bp[:, :, :k], sb.cuda(), c2, *args)
    assert torch.equal(c, c2)


@pytest.mark.parametrize("raw", [[0, -5, 9, 4, 12], [-7, 3, 3, 100, 2], [9, 2, 2, 2, 2], [12, 99, 99, -1, 5]])
def test_grouped_offsets_are_held_to_the_rows(cm, raw):
    """Offsets outside 0..n or out of order are held to that range and order."""
    n, k, m = 12, 256, 130
    a, sa, b, sb = operands(21, n, k, m, groups=4)
    ends = np.maximum.accumulate(np.clip(raw, 0, n)).tolist()
    want, mag = grouped_want(a, sa, b, sb, ends, -3.0)
    c = torch.full((n, m), -3.0, device="cuda")
    cm.MatmulKernelFp8Grouped(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, torch.tensor(raw, dtype=torch.int32, device="cuda"), 4, n, k, m)
    check_product(c.cpu(), want, mag, k, F32)


def test_grouped_shared_weights(cm):
    """A group stride of 0: every group uses the same weights, so the result is the dense product's."""
    n, k, m = 300, 512, 256
    a, sa, b, sb = operands(22, n, k, m)
    dev = [t.cuda() for t in (a, sa, b, sb)]
    c1, c2 = torch.empty(n, m, device="cuda"), torch.empty(n, m, device="cuda")
    cm.MatmulKernelFp8(*dev, c1, n, k, m)
    off = torch.tensor([0, 100, 100, 263, 300], dtype=torch.int32, device="cuda")
    cm.MatmulKernelFp8Grouped(*dev, c2, off, 4, n, k, m, ldb=k, b_group_stride=0, b_scale_ld=up(k), b_scale_group_stride=0)
    want, mag = product64(a, sa, b, sb)
    check_product(c1.cpu(), want, mag, k, F32)
    check_product(c2.cpu(), want, mag, k, F32)


# ---- as they are used ---------------------------------------------------------------------------------
class Block:
    """norm -> projection -> norm -> experts -> quantisation, on buffers of its own."""

    def __init__(self, cm, n, d, h, groups, seed):
        self.cm, self.n, self.d, self.h, self.groups = cm, n, d, h, groups
        e = lambda *s, t=BF16: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
        self.x, self.r = values(seed, n, d).to(BF16).cuda(), values(seed + 1, n, d).to(BF16).cuda()
        self.w1, self.w2 = ((1 + 0.1 * values(seed + i, d)).to(BF16).cuda() for i in (2, 3))
        wp, we = (torch.randn(d, d) * 0.05).to(BF16).cuda(), (torch.randn(groups, h, d) * 0.05).cuda()
        self.p, self.ps = e(d, d, t=E4), e(up(d), up(d), t=F32)
        self.e, self.es = e(groups, h, d, t=E4), e(groups, up(h), up(d), t=F32)
        cm.QuantKernelFp8(wp, self.p, self.ps, d, d, block_rows=128)
        cm.QuantKernelFp8(we, self.e, self.es, h, d, groups, block_rows=128)
        self.r1, self.r2, self.q1, self.q2 = e(n, d), e(n, d), e(n, d, t=E4), e(n, d, t=E4)
        self.s1, self.s2, self.y = e(up(d), n, t=F32), e(up(d), n, t=F32), e(n, d)
        self.z, self.zq, self.zs = e(n, h), e(n, h, t=E4), e(up(h), n, t=F32)
        cuts = sorted((torch.rand(groups - 1, generator=torch.Generator().manual_seed(seed)) * n).int().tolist())
        self.ends = [0, *cuts, n]
        self.off = torch.tensor(self.ends, dtype=torch.int32, device="cuda")

    def run(self, stream):
        cm, n, d, h = self.cm, self.n, self.d, self.h
        cm.RmsNormKernelFp8(self.x, self.w1, self.q1, self.s1, n, d, resid=self.r, resid_out=self.r1, stream=stream)
        cm.MatmulKernelFp8(self.q1, self.s1, self.p, self.ps, self.y, n, d, d, stream=stream)
        cm.RmsNormKernelFp8(self.y, self.w2, self.q2, self.s2, n, d, resid=self.r1, resid_out=self.r2, stream=stream)
        cm.MatmulKernelFp8Grouped(self.q2, self.s2, self.e, self.es, self.z, self.off, self.groups, n, d, h, stream=stream)
        cm.QuantKernelFp8(self.z, self.zq, self.zs, n, h, stream=stream)

    def outputs(self):
        return [t.clone() if t.dtype != E4 else t.view(torch.uint8).clone() for t in (self.r1, self.y, self.r2, self.z, self.zq, self.zs)]

    def check(self):
        """Each step from the inputs that it was given, in 64 bits."""
        c = lambda t: t.cpu()  # noqa: E731
        want, mag = product64(c(self.q1), c(self.s1), c(self.p), c(self.ps))
        check_product(c(self.y), want, mag, self.d, BF16)
        h = c(self.y).double() + c(self.r1).double()
        y2 = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * c(self.w2).double()
        s = expand(self.s2, self.n, self.d, 1)
        err = (c(self.q2).double() * s - y2).abs()
        assert (err <= torch.maximum(HALF_STEP[E4] * y2.abs(), HALF_SUBNORMAL[E4] * s) + 32 * U * y2.abs()).all()
        want, mag = grouped_want(c(self.q2), c(self.s2), c(self.e), c(self.es), self.ends, 0.0)
        check_product(c(self.z), want, mag, self.d, BF16)
        want_q, want_s = plain_quant(c(self.z).float(), E4, 1)
        assert torch.equal(c(self.zq).float(), want_q) and torch.equal(c(self.zs), want_s.t())


@pytest.mark.parametrize("n,d,h,groups", [(1, 512, 256, 4), (37, 1000, 300, 6), (700, 640, 384, 5)])
def test_a_block_of_them(cm, n, d, h, groups):
    b = Block(cm, n, d, h, groups, 100 + n)
    torch.cuda.synchronize()
    b.run(torch.cuda.current_stream())
    torch.cuda.synchronize()
    b.check()
    first = b.outputs()
    for _ in range(5):
        b.run(torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, b.outputs()))      # no order of additions changes


def test_two_blocks_on_two_streams_and_captured(cm):
    """Two captured graphs, replayed on two streams at once with changed inputs."""
    blocks = [Block(cm, 50, 1000, 300, 5, 300), Block(cm, 400, 512, 256, 3, 400)]
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    graphs = []
    for b, s in zip(blocks, streams):
        b.run(s)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.run(s)
        graphs.append(g)
    for round_ in range(3):
        for b in blocks:
            b.x.copy_(values(500 + round_, b.n, b.d))
            for t in (b.r1, b.y, b.r2, b.z):
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for b in blocks:
            b.check()


@pytest.mark.parametrize("n,d,h,groups", [(5, 512, 264, 3), (90, 1000, 520, 6), (1100, 640, 384, 4)])
def test_a_feed_forward_block_of_experts(cm, n, d, h, groups):
    """norm + quantise, grouped product, activation (in Q8.8, by the framework's own kernel), quantise, grouped product, on
    one stream; each step is checked from the inputs that it was given."""
    e = lambda *s, t: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    x, r, w = values(n, n, d).to(BF16).cuda(), values(n + 1, n, d).to(BF16).cuda(), (1 + 0.1 * values(n + 2, d)).to(BF16).cuda()
    gen = torch.Generator().manual_seed(n + 3)
    up_w, down_w = (torch.randn(groups, h, d, generator=gen) * 0.05).cuda(), (torch.randn(groups, d, h, generator=gen) * 0.05).cuda()
    u, us, v, vs = e(groups, h, d, t=E4), e(groups, up(h), up(d), t=F32), e(groups, d, h, t=E4), e(groups, up(d), up(h), t=F32)
    cm.QuantKernelFp8(up_w, u, us, h, d, groups, block_rows=128)
    cm.QuantKernelFp8(down_w, v, vs, d, h, groups, block_rows=128)
    ends = [0, *sorted((torch.rand(groups - 1, generator=gen) * n).int().tolist()), n]
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    q, s, h1, out, r1 = e(n, d, t=E4), e(up(d), n, t=F32), e(n, h, t=Q88), e(n, d, t=BF16), e(n, d, t=BF16)
    h2, hq, hs = e(n, h, t=Q88), e(n, h, t=E4), e(up(h), n, t=F32)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    cm.RmsNormKernelFp8(x, w, q, s, n, d, resid=r, resid_out=r1, stream=stream)
    cm.MatmulKernelFp8Grouped(q, s, u, us, h1, off, groups, n, d, h, stream=stream)
    cm.VectorOPKernel(h1, h1, h2, n * h, cm.OP_RELU, stream=stream)
    cm.QuantKernelFp8(h2, hq, hs, n, h, stream=stream)
    cm.MatmulKernelFp8Grouped(hq, hs, v, vs, out, off, groups, n, h, d, stream=stream)
    stream.synchronize()
    c = lambda t: t.cpu()  # noqa: E731
    want, mag = grouped_want(c(q), c(s), c(u), c(us), ends, 0.0)
    check_product(c(h1), want, mag, d, Q88)
    assert torch.equal(h2, h1.clamp_min(0)) and (h2 > 0).any()
    want_q, want_s = plain_quant(real(c(h2)).float(), E4, 1)
    assert torch.equal(c(hq).float(), want_q) and torch.equal(c(hs), want_s.t())
    want, mag = grouped_want(c(hq), c(hs), c(v), c(vs), ends, 0.0)
    check_product(c(out), want, mag, h, BF16)


def test_synchronous_entries_report(cm):
    """The entries without a stream return after the work, and refuse tensors that are too small."""
    a, sa, b, sb = (t.cuda() for t in operands(33, 5, 256, 130))
    c = torch.empty(5, 130, device="cuda")
    cm.MatmulKernelFp8(a, sa, b, sb, c, 5, 256, 130)
    with pytest.raises(ValueError):
        cm.MatmulKernelFp8(a, sa, b, sb, c, 6, 256, 130)
    with pytest.raises(ValueError):
        cm.MatmulKernelFp8(a, sa, b.t(), sb, c, 5, 256, 130)
    with pytest.raises(ValueError):
        cm.MatmulKernelFp8(a.flatten()[:-1], sa, b, sb, c, 5, 256, 130)
    with pytest.raises(TypeError):
        cm.MatmulKernelFp8(a, sa, b, sb, c.double(), 5, 256, 130)
    with pytest.raises(TypeError):
        cm.MatmulKernelFp8(a, sa.half(), b, sb, c, 5, 256, 130)
    with pytest.raises(TypeError):
        cm.MatmulKernelFp8(a, sa, b, sb, c, 5, 256, 130, a_fmt=cm.F8_E5M2)
    with pytest.raises(cm.CormorantError):
        cm.QuantKernelFp8(c, a, sa, 5, 130, block_rows=64)


@pytest.mark.parametrize("n,k,m", [(1, 4096, 256), (300, 512, 256)])
def test_first_call_of_a_new_thread(cm, n, k, m):
    """A thread that has not used the GPU yet may begin with a product."""
    import threading
    a, sa, b, sb = (t.cuda() for t in operands(n, n, k, m))
    want, c, failed = torch.empty(n, m, device="cuda"), torch.empty(n, m, device="cuda"), []
    cm.MatmulKernelFp8(a, sa, b, sb, want, n, k, m)

    def first():
        try:
            cm.MatmulKernelFp8(a, sa, b, sb, c, n, k, m)
        except BaseException as e:
            failed.append(e)

    t = threading.Thread(target=first)
    t.start()
    t.join()
    assert not failed, failed
    assert torch.equal(c, want)


FIRST_CALLS = """
import sys, threading
import torch
import cormorant_b200 as cm
sys.path.insert(0, "tests")
import test_gpu_fp8 as T
cm.init("0")
sizes = [(1, 4096, 256), (70, 512, 4096), (300, 1000, 1001), (1100, 512, 1300), (3000, 256, 2304)]
data = [[v.cuda() for v in T.operands(n, n, k, m)] for n, k, m in sizes]
out = [[torch.empty(n, m, device="cuda") for n, k, m in sizes] for _ in range(4)]
torch.cuda.synchronize()
ready, failed = threading.Barrier(4), []
def calls(i):
    stream = torch.cuda.Stream()
    ready.wait()
    try:
        for j in range(len(sizes)):
            j = (i + j) % len(sizes)
            cm.MatmulKernelFp8(*data[j], out[i][j], *sizes[j], stream=stream)
        stream.synchronize()
    except BaseException as e:
        failed.append(e)
threads = [threading.Thread(target=calls, args=(i,)) for i in range(4)]
for t in threads: t.start()
for t in threads: t.join()
assert not failed, failed
assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(o, out[0]))
for d, (n, k, m), c in zip(data, sizes, out[0]):
    T.check_product(c.cpu(), *T.product64(*(v.cpu() for v in d)), k, T.F32)
print("done")
"""


def test_first_calls_from_several_threads():
    """A process whose first calls of every tile come from four threads at once."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]


# ---- every tile ------------------------------------------------------------------------------------------
# The product's tile is chosen by size; which one a size takes is worked out here from the table in its source, so that
# a change of the rule shows as a test that no longer reaches the tile it names.
TILES = ["16", "32", "64", "256x128", "256x256"]


def tile_of(n, k, m, groups=0):
    import re
    from pathlib import Path
    source = (Path(__file__).resolve().parent.parent / "cormorant_b200" / "csrc" / "cm_fp8_gemm.cu").read_text()
    table = re.search(r"kinds\[\] = \{\s*(.*?)\};", source, re.S).group(1)
    kinds = [tuple(map(int, t.split(","))) for t in re.findall(r"\{([\d, ]+)\}", table)]
    assert len(kinds) == len(TILES)
    sms, costs = torch.cuda.get_device_properties(0).multi_processor_count, []
    for tokens, weights, ctas, block, out in kinds:
        rows = min(n, n // tokens + (groups + 1) // 2 + 1) if groups else -(-n // tokens)
        tiles, at_once = rows * -(-m // weights), sms // ctas
        costs.append(-(-tiles // at_once) * (up(k) * block + out))
    return TILES[costs.index(min(costs))]


@pytest.mark.parametrize("tile,n,k,m", [("16", 40, 640, 300), ("32", 90, 512, 4096), ("64", 200, 1000, 4096), ("256x128", 520, 300, 2050),
                                        ("256x256", 600, 512, 4224)])
def test_matmul_nan_and_infinity_stay_where_they_are(cm, tile, n, k, m):
    assert tile_of(n, k, m) == tile
    a, sa, b, sb = operands(9, n, k, m)
    want, mag = product64(a, sa, b, sb)
    ai, bi, sa = a.view(torch.uint8).clone(), b.view(torch.uint8).clone(), sa.clone()
    bad_rows, bad_cols = [1, n // 2, n - 1], [0, m // 2 + 1, m - 1]
    ai[1, 130], sa[1, n // 2], sa[up(k) - 1, n - 1] = 0x7F, float("nan"), float("inf")
    bi[bad_cols, k - 1] = 0xFF
    c = torch.empty(n, m, device="cuda")
    cm.MatmulKernelFp8(ai.view(E4).cuda(), sa.cuda(), bi.view(E4).cuda(), sb.cuda(), c, n, k, m)
    got = c.cpu()
    rows, cols = torch.ones(n, dtype=torch.bool), torch.ones(m, dtype=torch.bool)
    rows[bad_rows], cols[bad_cols] = False, False
    assert not torch.isfinite(got[~rows]).any() and torch.isnan(got[:, ~cols]).all()
    err = (got.double() - want).abs()
    assert (err <= (264 + 2 * up(k)) * U * mag + half(F32) * want.abs())[rows][:, cols].all()


# A group's last tile reads the rows behind it, which are another group's or no group's: NaN there stays there.
@pytest.mark.parametrize("tile,sizes,k,m", [("16", [11, 0, 29, 10], 300, 300), ("32", [50, 0, 50], 300, 3000), ("64", [70, 1, 100, 0, 129], 300, 2000),
                                            ("256x128", [700, 0, 800], 300, 2600), ("256x256", [300, 257, 0, 543], 300, 2040)])
def test_grouped_nan_stays_in_its_rows(cm, tile, sizes, k, m):
    ends = [3]
    for v in sizes:
        ends.append(ends[-1] + v)
    n = ends[-1] + 5
    assert tile_of(n, k, m, len(sizes)) == tile
    a, sa, b, sb = operands(k + m, n, k, m, groups=len(sizes))
    want, mag = grouped_want(a, sa, b, sb, ends, 0.0)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[: ends[0]] = bad[ends[-1]:] = True                                # no group's rows
    for i in ends[1:-1]:
        bad[i] = True                                                      # the first row of each group but one
    ai, sa = a.view(torch.uint8).clone(), sa.clone()
    ai[bad], sa[:, bad] = 0x7F, float("nan")
    c = torch.full((n, m), -3.0, device="cuda")
    cm.MatmulKernelFp8Grouped(ai.view(E4).cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, torch.tensor(ends, dtype=torch.int32, device="cuda"), len(sizes), n, k, m)
    got = c.cpu()
    assert (got[: ends[0]] == -3).all() and (got[ends[-1]:] == -3).all()
    inside = torch.zeros(n, dtype=torch.bool)
    inside[ends[0]: ends[-1]] = True
    assert torch.isnan(got[inside & bad]).all()
    err = (got.double() - want).abs()
    assert (err <= (264 + 2 * up(k)) * U * mag + half(F32) * want.abs())[inside & ~bad].all()


# Rows of c that start on 16-byte boundaries leave the wide tiles in whole 16-byte pieces.
@pytest.mark.parametrize("t", [F32, F16, BF16, Q88])
@pytest.mark.parametrize("tile,n,k,m", [("256x256", 600, 512, 4232), ("256x256", 1300, 300, 2632), ("256x128", 520, 300, 2056), ("256x128", 1100, 512, 1304)])
def test_matmul_aligned_output_rows(cm, tile, n, k, m, t):
    assert tile_of(n, k, m) == tile and m * t.itemsize % 16 == 0
    a, sa, b, sb = operands(n + m, n, k, m, E5 if t == F16 else E4, E4)
    want, mag = product64(a, sa, b, sb)
    c = torch.full((n + 2, m), -3, dtype=t, device="cuda")
    cm.MatmulKernelFp8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c[1:], n, k, m)
    check_product(c[1: n + 1].cpu(), want, mag, k, t)
    assert (c[0] == -3).all() and (c[n + 1] == -3).all()


@pytest.mark.parametrize("t", [F32, F16, BF16, Q88])
@pytest.mark.parametrize("tile,sizes,k,m", [("256x256", [300, 257, 0, 543], 300, 2040), ("256x256", [1, 1500, 999], 300, 2600), ("256x128", [700, 0, 800], 300, 2600)])
def test_grouped_aligned_output_rows(cm, tile, sizes, k, m, t):
    ends = [0]
    for v in sizes:
        ends.append(ends[-1] + v)
    n = ends[-1]
    assert tile_of(n, k, m, len(sizes)) == tile and m * t.itemsize % 16 == 0
    a, sa, b, sb = operands(k + m, n, k, m, groups=len(sizes))
    want, mag = grouped_want(a, sa, b, sb, ends, 0.0)
    c = torch.full((n + 1, m), -3, dtype=t, device="cuda")
    cm.MatmulKernelFp8Grouped(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, torch.tensor(ends, dtype=torch.int32, device="cuda"), len(sizes), n, k, m)
    check_product(c[:n].cpu(), want, mag, k, t)
    assert (c[n] == -3).all()


@pytest.mark.parametrize("pair", [("16", "256x256"), ("256x128", "64"), ("256x256", "256x128"), ("32", "16")])
def test_every_tile_captured_on_two_streams(cm, pair):
    """Two graphs of a dense and a grouped product each, replayed side by side with changed inputs."""
    sizes = {"16": (40, 640, 300), "32": (90, 512, 4096), "64": (200, 1000, 4096), "256x128": (520, 300, 2050), "256x256": (600, 512, 4224)}
    grouped = {"16": ([11, 0, 29, 10], 300, 300), "32": ([50, 0, 50], 300, 3000), "64": ([70, 1, 100, 0, 129], 300, 2000),
               "256x128": ([700, 0, 800], 300, 2600), "256x256": ([300, 257, 0, 543], 300, 2040)}
    work = []
    for tile in pair:
        n, k, m = sizes[tile]
        gs, gk, gm = grouped[tile]
        ends = np.cumsum([0, *gs]).tolist()
        assert tile_of(n, k, m) == tile and tile_of(ends[-1], gk, gm, len(gs)) == tile
        dev = lambda ops: [v.cuda() for v in ops]  # noqa: E731
        d, g = dev(operands(n, n, k, m)), dev(operands(gm, ends[-1], gk, gm, groups=len(gs)))
        off = torch.tensor(ends, dtype=torch.int32, device="cuda")
        c, gc, s = torch.empty(n, m, dtype=BF16, device="cuda"), torch.empty(ends[-1], gm, device="cuda"), torch.cuda.Stream()

        def run(d=d, g=g, c=c, gc=gc, off=off, s=s, n=n, k=k, m=m, gs=gs, gk=gk, gm=gm, ends=ends):
            cm.MatmulKernelFp8(*d, c, n, k, m, stream=s)
            cm.MatmulKernelFp8Grouped(*g, gc, off, len(gs), ends[-1], gk, gm, stream=s)

        torch.cuda.synchronize()
        run()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run()
        work.append((graph, s, d, g, c, gc, k, gk, ends))
    for change in range(2):
        for _, _, d, g, c, gc, *_ in work:
            d[1].mul_(1 + change)
            g[3].mul_(1 + change)
            c.fill_(float("nan"))
            gc.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, s, *_ in work:
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for _, _, d, g, c, gc, k, gk, ends in work:
            check_product(c.cpu(), *product64(*(v.cpu() for v in d)), k, BF16)
            check_product(gc.cpu(), *grouped_want(*(v.cpu() for v in g), ends, 0.0), gk, F32)


@pytest.mark.parametrize("n,k,m,groups", [(5, 256, 130, 4), (300, 512, 260, 3), (1100, 300, 2040, 4)])
@pytest.mark.parametrize("layout", ["rows side by side", "odd gap", "16-byte gap"])
def test_grouped_weights_at_any_group_stride(cm, n, k, m, groups, layout):
    """Groups whose rows lie between each other's, and groups that lie no whole number of rows apart."""
    a, sa, b, sb = operands(n, n, k, m, groups=groups)
    ends = [n * i // groups for i in range(groups + 1)]
    want, mag = grouped_want(a, sa, b, sb, ends, 0.0)
    k16 = (k + 15) // 16 * 16
    ld, gs = (groups * k16, k16) if layout == "rows side by side" else (k16, m * k16 + (16 if layout == "16-byte gap" else 7))
    buf = torch.full(((groups - 1) * gs + (m - 1) * ld + k16,), 0x7F, dtype=torch.uint8, device="cuda")
    view = buf.as_strided((groups, m, k), (gs, ld, 1))
    view.copy_(b.view(torch.uint8))
    c = torch.full((n, m), -3.0, device="cuda")
    cm.MatmulKernelFp8Grouped(a.cuda(), sa.cuda(), view.view(E4), sb.cuda(), c, torch.tensor(ends, dtype=torch.int32, device="cuda"), groups, n, k, m)
    check_product(c.cpu(), want, mag, k, F32)


@pytest.mark.parametrize("n,k,m", [(3, 128, 130), (600, 512, 4224)])
def test_matmul_q88_of_nan_and_infinity(cm, n, k, m):
    a, sa, b, sb = operands(n, n, k, m)
    want, mag = product64(a, sa, b, sb)
    sa = sa.clone()
    sa[0, 0], sa[0, 1] = float("nan"), float("inf")
    c = torch.full((n, m), 77, dtype=Q88, device="cuda")
    cm.MatmulKernelFp8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), c, n, k, m)
    got, first = c.cpu(), (a[1, :128].double() @ b[:, :128].double().t())
    assert (got[0] == 0).all()
    assert torch.equal(got[1], torch.where(first > 0, 32767, torch.where(first < 0, -32768, 0)).to(Q88))
    check_product(got[2:], want[2:], mag[2:], k, Q88)


def test_a_refused_allocation_is_not_the_next_calls_error(cm):
    """A product whose aligned copies would take 1 TB is answered with CM_ENOMEM, and the next call has a result of its own."""
    n, k, m, groups = 1, 1000, 1 << 20, 1024
    a, sa, b, sb = (t.cuda() for t in operands(3, 40, 256, 130))
    want, c = torch.empty(40, 130, device="cuda"), torch.empty(40, 130, device="cuda")
    cm.MatmulKernelFp8(a, sa, b, sb, want, 40, 256, 130)
    w = torch.zeros(groups - 1 + m * k, dtype=torch.uint8, device="cuda")           # the groups' weights overlap: one byte apart
    big = (torch.zeros(n, k, dtype=E4, device="cuda"), torch.zeros(up(k), n, device="cuda"), w.view(E4), torch.zeros(up(m), up(k), device="cuda"),
           torch.zeros(n, m, device="cuda"), torch.zeros(groups + 1, dtype=torch.int32, device="cuda"), groups, n, k, m)
    with pytest.raises(cm.CormorantError, match="memory"):
        cm.MatmulKernelFp8Grouped(*big, ldb=k, b_group_stride=1, b_scale_ld=up(k), b_scale_group_stride=0)
    cm.MatmulKernelFp8(a, sa, b, sb, c, 40, 256, 130)
    assert torch.equal(c, want)
    q, s = torch.empty(40, 130, dtype=E4, device="cuda"), torch.empty(2, 40, device="cuda")
    with pytest.raises(cm.CormorantError, match="memory"):
        cm.MatmulKernelFp8Grouped(*big, ldb=k, b_group_stride=1, b_scale_ld=up(k), b_scale_group_stride=0)
    cm.QuantKernelFp8(c, q, s, 40, 130)
    torch.cuda.synchronize()


FIRST_CAPTURED = """
import sys
import torch
import cormorant_b200 as cm
sys.path.insert(0, "tests")
import test_gpu_fp8 as T
cm.init("0")
sizes = [(1, 4096, 256), (70, 512, 4096), (300, 1000, 1001), (1100, 512, 1300), (3000, 250, 2304)]
data = [[v.cuda() for v in T.operands(n, n, k, m)] for n, k, m in sizes]
out = [torch.empty(n, m, device="cuda") for n, k, m in sizes]
x, q, s = T.values(1, 37, 1000).cuda(), torch.empty(37, 1000, dtype=T.E4, device="cuda"), torch.empty(8, 37, device="cuda")
torch.cuda.synchronize()
graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(graph, stream=stream):
    for d, size, c in zip(data, sizes, out):
        cm.MatmulKernelFp8(*d, c, *size, stream=stream)
    cm.QuantKernelFp8(x, q, s, 37, 1000, stream=stream)
for _ in range(2):
    for c in out:
        c.fill_(float("nan"))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for d, (n, k, m), c in zip(data, sizes, out):
        T.check_product(c.cpu(), *T.product64(*(v.cpu() for v in d)), k, T.F32)
    assert torch.equal(q.float().cpu(), T.plain_quant(x.cpu(), T.E4, 1)[0])
print("done")
"""


def test_first_calls_captured():
    """A process whose first calls are recorded into a graph, one with operands that are copied into aligned rows."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_CAPTURED], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
