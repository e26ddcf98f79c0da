"""Rows to 8-bit integers (eco_quant_rows_forward) and the inner product of such rows (eco_inner_product_i8_forward) against
their definitions, on both backends.

The integers are exact: 127 |x| has 31 bits and max |x| has 24, so a quotient that is not a tie is further than 2^-32 of itself
from one and numpy's float64 quotient rounds to the same integer.  A product's sum is exact, the conversion to fp32, two
multiplications and an addition round by 2^-24 each: 6 * 2^-24 of |sum sx sw| + |bias| bounds them; SiLU's slope is below 1.1 and
its exponential off by (4 + |v|) fp32 roundings; then half a step of the output's type."""
import numpy as np
import pytest

from eco_amd import hip
from tests.test_group_norm import U32, UNIT, from_bits, store, to_bits, value

TYPES = pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])


# ---- rows to integers ------------------------------------------------------------------------------------------------------
def quant_reference(x):
    """(q, scale) of float32 rows."""
    with np.errstate(all="ignore"):
        top = np.abs(x).max(axis=1, keepdims=True)
        fine = np.isfinite(x).all(axis=1, keepdims=True)
        quotient = x.astype(np.float64) * 127.0 / top.astype(np.float64)
        q = np.where(fine & (top > 0), np.rint(np.where(np.isfinite(quotient), quotient, 0.0)), 0.0)
        scale = np.where(fine, top / np.float32(127.0), np.float32(np.nan))
    return q.astype(np.int8), scale[:, 0].astype(np.float32)


def run_quant(be, x, dt, xgap=0, qgap=0, xshift=0, qshift=0):
    m, k = x.shape
    flat = np.full(xshift + m * (k + xgap), 9.0, np.float32)
    flat[xshift:].reshape(m, k + xgap)[:, :k] = x
    size = 4 if dt == hip.DT_F32 else 2
    dx, dq, ds = be.dev(store(flat, dt)), be.dev(np.full(qshift + m * (k + qgap), 99, np.int8)), be.dev(np.full(m + 1, 5.0, np.float32))
    p = be.alloc.ptr
    be.lib.quant_rows_forward(p(dx) + xshift * size, dt, p(dq) + qshift, p(ds), m, k, ldx=k + xgap if xgap else 0,
                              ldq=k + qgap if qgap else 0)
    q = be.host(dq, (qshift + m * (k + qgap),))
    assert (q[:qshift] == 99).all() and (q[qshift:].reshape(m, k + qgap)[:, k:] == 99).all()
    scale = be.host(ds, (m + 1,))
    assert scale[m] == 5.0
    want_q, want_s = quant_reference(x)
    got = q[qshift:].reshape(m, k + qgap)[:, :k]
    assert np.array_equal(got, want_q), np.argwhere(got != want_q)[:5]
    assert np.array_equal(scale[:m], want_s, equal_nan=True)


def rows(rng, m, k, dt):
    x = rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))
    return value(store(x.astype(np.float32), dt), dt)


@TYPES
@pytest.mark.parametrize("m,k", [(1, 1), (5, 3), (7, 8), (3, 64), (9, 100), (4, 128), (6, 511), (3, 512), (5, 520), (2, 1000),
                                 (2, 2049), (1, 4100), (2, 9000), (1, 20000), (70, 16), (33, 24)])
def test_quant_matches_the_exact_quotient(backend, m, k, dt):
    run_quant(backend, rows(np.random.default_rng(m + k), m, k, dt), dt)


@TYPES
@pytest.mark.parametrize("xgap,qgap,xshift,qshift", [(8, 8, 0, 0), (8, 0, 8, 0), (3, 0, 0, 0), (0, 5, 0, 1), (0, 0, 1, 4), (16, 16, 16, 16)])
def test_quant_strides_alignment_and_guards(backend, dt, xgap, qgap, xshift, qshift):
    for k in (40, 700):
        run_quant(backend, rows(np.random.default_rng(k), 6, k, dt), dt, xgap, qgap, xshift, qshift)


@TYPES
def test_quant_ties_and_their_neighbours(backend, dt):
    """Quotients of exactly k + 1/2 (to the even integer) and the type's next values on either side of them."""
    for top in (127.0, 254.0, 63.5, 1.9375, 2.0 ** -100 * 127, 3.0e38, 1.0):
        top = float(value(store(np.float32([top]), dt), dt)[0])
        ties = np.float32((np.arange(127) + 0.5) * (top / 127.0))
        ties = value(store(ties, dt), dt)
        if dt == hip.DT_F32:
            near = np.concatenate([ties, np.nextafter(ties, np.float32(0)), np.nextafter(ties, np.float32(np.inf))])
        else:
            b = to_bits(ties)
            near = np.concatenate([ties, from_bits((b - 1).astype(np.uint16)), from_bits((b + 1).astype(np.uint16))])
        near = near[np.abs(near) <= top]
        x = np.concatenate([near, -near, [top]]).astype(np.float32)
        run_quant(backend, np.stack([x, -x]), dt)


@TYPES
def test_quant_special_rows(backend, dt):
    """Zeros (of both signs), NaN, infinities, the largest and the smallest values of the type."""
    x = rows(np.random.default_rng(1), 12, 72, dt)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 5] = np.nan
    x[3, 71] = np.inf
    x[4, 0] = -np.inf
    x[5] = 0.0
    x[5, 9] = -1e-40                      # subnormal
    x[6] *= np.float32(1e-38)
    x[7, 3] = value(store(np.float32([3.38e38]), dt), dt)[0]
    x[8] = np.float32(2.0 ** -133)
    x[9, :] = -1.0
    x = value(store(x, dt), dt)
    run_quant(backend, x, dt)


def test_quant_nothing_to_do_and_refusals(backend):
    lib = backend.lib
    lib.quant_rows_forward(None, hip.DT_F32, None, None, 0, 8)
    x, q, s = backend.dev(np.ones(64, np.float32)), backend.dev(np.full(64, 99, np.int8)), backend.dev(np.full(8, 5.0, np.float32))
    p = backend.alloc.ptr
    ok = dict(x=p(x), dt=hip.DT_F32, q=p(q), scale=p(s), m=4, k=8)
    for kw in (dict(dt=2), dict(m=-1), dict(k=0), dict(x=None), dict(q=None), dict(scale=None), dict(ldx=7), dict(ldq=7),
               dict(ldx=-8), dict(x=p(x) + 2), dict(ldx=2 ** 62), dict(ldq=2 ** 62), dict(k=2 ** 40), dict(k=2 ** 30 + 1, ldx=2 ** 31), dict(m=2 ** 31)):
        with pytest.raises(hip.EcoError, match="quant_rows"):
            lib.quant_rows_forward(**{**ok, **kw})
    assert (backend.host(q, (64,)) == 99).all() and (backend.host(s, (8,)) == 5.0).all()


# ---- the product -----------------------------------------------------------------------------------------------------------
def operand(be, a, gap, shift, fill=113):
    """int8 rows `gap` bytes apart, the first `shift` bytes into its buffer; what lies between must not be summed."""
    m, k = a.shape
    flat = np.full(shift + m * (k + gap) - gap, fill, np.int8)
    np.lib.stride_tricks.as_strided(flat[shift:], (m, k), (k + gap, 1))[...] = a
    return be.dev(flat)


class Product:
    def __init__(self, be, m, n, k, dt, act=hip.ACT_NONE, bias=True, gaps=(0, 0, 0), shifts=(0, 0, 0), seed=0, num_cu=None,
                 extreme=False, scale_shift=0):
        rng = np.random.default_rng(seed)
        self.be, self.m, self.n, self.k, self.dt, self.act, self.gaps, self.shifts = be, m, n, k, dt, act, gaps, shifts
        if extreme:
            self.x, self.w = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
        else:
            self.x, self.w = (rng.integers(-128, 128, sh).astype(np.int8) for sh in ((m, k), (n, k)))
        self.sx = (0.01 + rng.random(m)).astype(np.float32)
        self.sw = ((0.01 + rng.random(n)) / (5000 * np.sqrt(k))).astype(np.float32)
        self.bias = rng.standard_normal(n).astype(np.float32) if bias else None
        self.plan = be.lib.inner_product_i8_plan(m, n, k, dt, num_cu)
        self.dx, self.dw = operand(be, self.x, gaps[0], shifts[0]), operand(be, self.w, gaps[1], shifts[1])
        # scales and bias `scale_shift` floats into their buffers: on a 4-byte boundary, no more
        self.scale_shift = scale_shift
        lead = np.full(scale_shift, 7.0, np.float32)
        self.dsx, self.dsw = be.dev(np.concatenate([lead, self.sx])), be.dev(np.concatenate([lead, self.sw]))
        self.db = be.dev(np.concatenate([lead, self.bias])) if bias else None
        self.total = shifts[2] + m * (n + gaps[2])
        self.dy = be.dev(store(np.full(self.total, 3.0, np.float32), dt))
        self.ws = be.empty((self.plan.ws_bytes // 4,), np.int32) if self.plan.ws_bytes else None

    def call(self, **kw):
        p = lambda h: None if h is None else self.be.alloc.ptr(h)  # noqa: E731
        size = 4 if self.dt == hip.DT_F32 else 2
        args = dict(act=self.act, ldx=self.k + self.gaps[0], ldw=self.k + self.gaps[1], ldy=self.n + self.gaps[2], workspace=p(self.ws))
        args.update(kw)
        f = 4 * self.scale_shift
        self.be.lib.inner_product_i8_forward(self.plan, p(self.dx) + self.shifts[0], p(self.dsx) + f, p(self.dw) + self.shifts[1],
                                             p(self.dsw) + f, p(self.db) + f if self.db is not None else None,
                                             p(self.dy) + self.shifts[2] * size, **args)

    def check(self):
        flat = value(self.be.host(self.dy, (self.total,)), self.dt)
        body = flat[self.shifts[2]:].reshape(self.m, self.n + self.gaps[2])
        assert (flat[: self.shifts[2]] == 3.0).all() and (body[:, self.n:] == 3.0).all()
        s = (self.x.astype(np.float64) @ self.w.astype(np.float64).T) * self.sx[:, None].astype(np.float64) * self.sw
        b = 0.0 if self.bias is None else self.bias.astype(np.float64)
        v, tol = s + b, 6 * U32 * (np.abs(s) + np.abs(b))
        if self.act == hip.ACT_RELU:
            v = np.maximum(v, 0.0)
        elif self.act == hip.ACT_SILU:
            y = v / (1.0 + np.exp(-v))
            tol = 1.1 * tol + 2 * U32 * (4 + np.abs(v)) * np.abs(y)
            v = y
        worst = np.abs(body[:, : self.n] - v) - (tol + UNIT[self.dt] * np.abs(v))
        assert worst.max() <= 0, (worst.max(), np.unravel_index(worst.argmax(), worst.shape))


def run_product(be, *a, **kw):
    case = Product(be, *a, **kw)
    case.call()
    case.check()


SIZES = [(1, 1, 1), (1, 16, 16), (1, 40, 512), (2, 33, 70), (3, 5, 129), (16, 16, 64), (17, 40, 100), (24, 64, 256), (31, 20, 48),
         (33, 33, 33), (64, 64, 64), (65, 70, 80), (100, 36, 160), (130, 129, 128), (200, 72, 31), (40, 300, 96)]


@TYPES
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_matches_the_formula(backend, m, n, k, dt):
    run_product(backend, m, n, k, dt, act=(hip.ACT_NONE, hip.ACT_RELU, hip.ACT_SILU)[(m + n + k) % 3], seed=m + n + k)


@TYPES
@pytest.mark.parametrize("gaps,shifts", [((16, 16, 8), (0, 0, 0)), ((16, 0, 0), (16, 32, 4)), ((1, 0, 1), (0, 0, 0)), ((0, 3, 0), (1, 2, 1)),
                                         ((0, 0, 2), (0, 5, 3)), ((8, 8, 4), (8, 8, 0))])
@pytest.mark.parametrize("m", [3, 70])
def test_product_strides_alignment_and_guards(backend, m, dt, gaps, shifts):
    run_product(backend, m, 48, 96, dt, gaps=gaps, shifts=shifts, act=hip.ACT_RELU)
    run_product(backend, m, 37, 83, dt, gaps=gaps, shifts=shifts, bias=False)


@TYPES
@pytest.mark.parametrize("m,n,k,shift", [(3, 40, 64, 1), (70, 72, 96, 1), (200, 136, 160, 3), (300, 264, 64, 2), (90, 37, 50, 1)])
def test_product_scales_on_any_boundary(backend, m, n, k, shift, dt):
    run_product(backend, m, n, k, dt, scale_shift=shift, act=hip.ACT_SILU)


@pytest.mark.parametrize("num_cu", [1, 5])
@pytest.mark.parametrize("m,n,k", [(5, 24, 700), (20, 40, 352), (40, 70, 288), (64, 33, 100), (90, 50, 640), (90, 56, 1040), (300, 260, 70), (200, 200, 512),
                                   (600, 520, 96)])
def test_product_plans_for_other_sizes_of_device(backend, m, n, k, num_cu):
    run_product(backend, m, n, k, hip.DT_F32, num_cu=num_cu, act=hip.ACT_SILU)


@pytest.mark.parametrize("m", [1, 40])
def test_product_of_the_lowest_values(backend, m):
    """-128 * -128 over long sums: the largest that 32 bits have to hold."""
    run_product(backend, m, 20, 2000, hip.DT_F32, extreme=True)


def test_product_of_a_row_with_scale_nan(backend):
    case = Product(backend, 5, 20, 64, hip.DT_F32)
    case.sx[2] = np.nan
    case.x[2] = 0
    case.dx, case.dsx = operand(backend, case.x, 0, 0), backend.dev(case.sx)
    case.call()
    y = backend.host(case.dy, (5, 20))
    assert np.isnan(y[2]).all() and np.isfinite(y[[0, 1, 3, 4]]).all()


def test_product_nothing_to_do(backend):
    p = backend.lib.inner_product_i8_plan(0, 8, 8, hip.DT_F32)
    backend.lib.inner_product_i8_forward(p, None, None, None, None, None, None)


@pytest.mark.parametrize("kw", [dict(m=-1), dict(n=0), dict(k=0), dict(k=hip.I8_MAX_K + 1), dict(m=2 ** 31), dict(n=2 ** 31), dict(n=2 ** 30 + 1), dict(m=2 ** 31 - 1, n=2 ** 30), dict(dt=2),
                                dict(num_cu=-1)], ids=lambda v: "-".join(f"{a}{b}" for a, b in v.items()))
def test_product_refused_plans(backend, kw):
    with pytest.raises(hip.EcoError, match="inner_product_i8"):
        backend.lib.inner_product_i8_plan(**{**dict(m=4, n=8, k=16, dt=hip.DT_F32), **kw})


def test_product_refused_launches(backend):
    """More channels than the plan takes; more tiles than a launch has (refused before anything is launched)."""
    with pytest.raises(hip.EcoError, match="channels"):
        backend.lib.inner_product_i8_plan(4, 2 ** 26 + 1, 16, hip.DT_F32)
    p = backend.lib.inner_product_i8_plan(64 << 13, 64 << 12, 1, hip.DT_F32)
    with pytest.raises(hip.EcoError, match="one launch"):
        backend.lib.inner_product_i8_forward(p, 16, 16, 16, 16, None, 16, workspace=16)


def test_product_refused_calls(backend):
    case = Product(backend, 4, 8, 16, hip.DT_F32)
    lib, p = backend.lib, backend.alloc.ptr
    for kw in (dict(act=3), dict(act=-1), dict(ldx=15), dict(ldw=15), dict(ldy=7), dict(ldx=-16), dict(ldx=2 ** 62), dict(ldw=2 ** 62),
               dict(ldy=2 ** 62)):
        with pytest.raises(hip.EcoError, match="inner_product_i8"):
            case.call(**kw)
    good = [p(case.dx), p(case.dsx), p(case.dw), p(case.dsw), None, p(case.dy)]
    for i in (0, 1, 2, 3, 5):
        bad = list(good)
        bad[i] = None
        with pytest.raises(hip.EcoError, match="null"):
            lib.inner_product_i8_forward(case.plan, *bad)
    with pytest.raises(hip.EcoError, match="aligned"):
        lib.inner_product_i8_forward(case.plan, *good[:5], good[5] + 2)
    other = lib.inner_product_i8_plan(4, 8, 16, hip.DT_F32)
    other.bm += 1
    with pytest.raises(hip.EcoError, match="plan"):
        lib.inner_product_i8_forward(other, *good)
    assert (backend.host(case.dy, (32,)) == 3.0).all()


@TYPES
def test_block_of_a_network(backend, dt):
    """The three operators as they are used: normalise and activate positions, quantise them and the weights, multiply."""
    be = backend
    rng = np.random.default_rng(5)
    n, s, c, cout, groups = 2, 45, 64, 40, 8
    lib, p = be.lib, be.alloc.ptr
    x = value(store(rng.standard_normal((n, s, c)).astype(np.float32), dt), dt)
    w = (rng.standard_normal((cout, c)) / 8).astype(np.float32)
    bias = rng.standard_normal(cout).astype(np.float32)
    dx, dw, db = be.dev(store(x, dt)), be.dev(w), be.dev(bias)
    h, y = be.empty((n * s * c,), np.float32 if dt == hip.DT_F32 else np.uint16), be.empty((n * s * cout,), np.float32 if dt == hip.DT_F32 else np.uint16)
    q, sq, qw, sw = be.empty((n * s * c,), np.int8), be.empty((n * s,)), be.empty((cout * c,), np.int8), be.empty((cout,))
    norm, prod = lib.group_norm_plan(n, s, c, groups, dt), lib.inner_product_i8_plan(n * s, cout, c, dt)
    ws = be.empty((max(norm.ws_bytes, prod.ws_bytes) // 4 + 1,))
    lib.quant_rows_forward(p(dw), hip.DT_F32, p(qw), p(sw), cout, c)
    lib.group_norm_forward(norm, p(dx), None, None, p(h), act=hip.ACT_SILU, workspace=p(ws))
    lib.quant_rows_forward(p(h), dt, p(q), p(sq), n * s, c)
    lib.inner_product_i8_forward(prod, p(q), p(sq), p(qw), p(sw), p(db), p(y), act=hip.ACT_RELU, workspace=p(ws))
    z = x.astype(np.float64).reshape(n, s, groups, -1)
    z = (z - z.mean(axis=(1, 3), keepdims=True)) / np.sqrt(z.var(axis=(1, 3), keepdims=True) + 1e-5)
    z = (z / (1 + np.exp(-z))).reshape(n * s, c)
    ref = np.maximum(z @ w.astype(np.float64).T + bias, 0.0)
    got = value(be.host(y, (n * s, cout)), dt).astype(np.float64)
    # half an integer step on either side of each of the c products, the norm's output rounded to dt, y rounded to dt
    step_x, step_w = np.abs(z).max(axis=1, keepdims=True) / 127, np.abs(w).max(axis=1) / 127
    tol = 0.5 * step_x * np.abs(w).sum(axis=1) + 0.5 * step_w * np.abs(z).sum(axis=1, keepdims=True) + 0.25 * c * step_x * step_w
    tol = (1 + 4 * UNIT[dt]) * tol + 2 * UNIT[dt] * (np.abs(z) @ np.abs(w).T) + UNIT[dt] * np.abs(ref) + 1e-5
    assert (np.abs(got - ref) <= tol).all()


# ---- on the device ----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@TYPES
@pytest.mark.parametrize("m,n,k", [(1, 400, 512), (1, 8192, 2048), (24, 5120, 1024), (32, 1000, 4096), (5000, 128, 128), (1003, 777, 1531),
                                   (700, 512, 2048), (2048, 1536, 512), (40, 64, 30000), (8, 16, hip.I8_MAX_K), (513, 769, 96), (4000, 257, 65)])
def test_product_device_sizes(hip_backend, m, n, k, dt):
    run_product(hip_backend, m, n, k, dt, act=hip.ACT_SILU)


@pytest.mark.gpu
def test_quant_device_sizes(hip_backend):
    for dt in (hip.DT_F32, hip.DT_BF16):
        for m, k in ((20000, 128), (3000, 500), (100, 16384), (3, 100001), (1, 4096)):
            run_quant(hip_backend, rows(np.random.default_rng(k), m, k, dt), dt)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(hip_backend):
    """The last rows of operands and results that pass 4 GiB."""
    import torch
    lib, stream = hip_backend.lib, torch.cuda.current_stream().cuda_stream
    k, n, m, ldx = 128, 64, 200, 1 << 25               # rows 32 MiB apart
    x = torch.zeros((m - 1) * ldx + k, dtype=torch.int8, device="cuda")
    xv = torch.as_strided(x, (m, k), (ldx, 1))
    xv.copy_(torch.randint(-128, 128, (m, k), device="cuda", dtype=torch.int8))
    w = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8)
    sx, sw = torch.rand(m, device="cuda"), torch.rand(n, device="cuda")
    y = torch.zeros(m, n, device="cuda")
    p = lib.inner_product_i8_plan(m, n, k, hip.DT_F32)
    ws = torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device="cuda")
    lib.inner_product_i8_forward(p, x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), None, y.data_ptr(), ldx=ldx,
                                 workspace=ws.data_ptr(), stream=stream)
    want = (xv.cpu().double() @ w.cpu().double().t()) * sx.cpu().double()[:, None] * sw.cpu().double()
    assert ((y.cpu().double() - want).abs() <= 8 * U32 * want.abs()).all()
    ldy = 1 << 23                                       # results' rows 32 MiB apart
    big = torch.zeros((m - 1) * ldy + n, device="cuda")
    dense = xv.contiguous()
    lib.inner_product_i8_forward(p, dense.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), None, big.data_ptr(), ldy=ldy,
                                 workspace=ws.data_ptr(), stream=stream)
    assert torch.equal(torch.as_strided(big, (m, n), (ldy, 1)), y)
    xq = torch.zeros((m - 1) * (ldx // 4) + k, device="cuda")
    xqv = torch.as_strided(xq, (m, k), (ldx // 4, 1))
    xqv.copy_(torch.randn(m, k, device="cuda"))
    q, s = torch.zeros((m - 1) * ldx + k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    lib.quant_rows_forward(xq.data_ptr(), hip.DT_F32, q.data_ptr(), s.data_ptr(), m, k, ldx=ldx // 4, ldq=ldx, stream=stream)
    want_q, want_s = quant_reference(xqv.cpu().numpy())
    assert np.array_equal(torch.as_strided(q, (m, k), (ldx, 1)).cpu().numpy(), want_q)
    assert np.array_equal(s.cpu().numpy(), want_s)


@pytest.mark.gpu
def test_quant_more_rows_than_one_launch_takes(hip_backend):
    """17 million rows that a workgroup each takes: 2^32 threads and more.  (Ones and a largest value per row: its integers are known.)"""
    import torch
    m, k = (1 << 24) + 77, 257
    x = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
    top = (torch.arange(m, device="cuda") % 126 + 2).bfloat16()
    x[:, 200] = -top
    q, s = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
    hip_backend.lib.quant_rows_forward(x.data_ptr(), hip.DT_BF16, q.data_ptr(), s.data_ptr(), m, k,
                                       stream=torch.cuda.current_stream().cuda_stream)
    assert torch.equal(s.cpu(), top.float().cpu() / 127.0)
    assert bool((q[:, 200] == -127).all())
    one = torch.round(127.0 / top.double()).to(torch.int8)
    assert bool((q[:, :200] == one[:, None]).all()) and bool((q[:, 201:] == one[:, None]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (70, 256, 4096), (600, 640, 512)])
def test_streams_and_graph_replays(hip_backend, m, n, k):
    """Quantise and multiply on two streams at once, then captured and replayed on new inputs: the eager bits each time."""
    import torch
    lib = hip_backend.lib
    p = lib.inner_product_i8_plan(m, n, k, hip.DT_BF16)
    w, sw = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8), torch.rand(n, device="cuda")

    class Buffers:
        def __init__(self):
            self.x = torch.empty(m, k, device="cuda")
            self.q = torch.empty(m, k, device="cuda", dtype=torch.int8)
            self.s, self.y = torch.empty(m, device="cuda"), torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
            self.ws = torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device="cuda")

        def call(self):
            stream = torch.cuda.current_stream().cuda_stream
            lib.quant_rows_forward(self.x.data_ptr(), hip.DT_F32, self.q.data_ptr(), self.s.data_ptr(), m, k, stream=stream)
            lib.inner_product_i8_forward(p, self.q.data_ptr(), self.s.data_ptr(), w.data_ptr(), sw.data_ptr(), None, self.y.data_ptr(),
                                         workspace=self.ws.data_ptr(), stream=stream)

    xs = [torch.randn(m, k, device="cuda") for _ in range(4)]
    want, sets = [], [Buffers() for _ in range(4)]
    for x in xs:
        sets[0].x.copy_(x)
        sets[0].call()
        want.append(sets[0].y.clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i, b in enumerate(sets):
        b.y.zero_()
        b.x.copy_(xs[i])
    torch.cuda.synchronize()
    for i, b in enumerate(sets):
        with torch.cuda.stream(streams[i % 2]):
            b.call()
    torch.cuda.synchronize()
    for i, b in enumerate(sets):
        assert torch.equal(b.y, want[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sets[0].call()
    for i in (2, 0, 3, 1, 2):
        sets[0].x.copy_(xs[i])
        sets[0].ws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(sets[0].y, want[i])
        assert float((xs[i] * 2).abs().sum()) > 0         # the program's own eager work between the replays
