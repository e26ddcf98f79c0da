"""Group norm with an activation over channels-last positions (eco_group_norm_forward) against its formula in 64 bits, on
both backends.

Tolerances, per value: half a step of the output's type (bf16 2^-8, fp32 2^-24, relative), plus 16 fp32 roundings of the sizes
that the formula passes through: (|x| + |mean| + mean|x|) * rstd * |gamma| and |beta|.  mean|x|, the group's mean magnitude, is for
the mean's own error: a partial sum of k values rounds by 2^-24 of itself, which is sqrt(k) mean|x| for values of both signs and
k |mean| for others; over a thread's up to 64 values, if every rounding went the same way, that is sum(sqrt(k))/64 = 5.3 mean|x|
or 32 |mean| (counted by |x| + |mean|, of which a value far from zero has both), and the joins of threads and chunks add at most
5 + 6 more sums of the same kind.  (A value near zero in a group of mean zero has no other part in its tolerance.)  A variance
is off by a few 2^-24 relative.  SiLU's slope is below 1.1, its exponential is off by (4 + |v|) fp32 roundings."""
import numpy as np
import pytest

from eco_amd import hip

U32 = 2.0 ** -24
UNIT = {hip.DT_F32: U32, hip.DT_BF16: 2.0 ** -8}
EPS = 1e-5


def to_bits(v):
    """float32 -> bf16 bits, nearest even (NaN kept)."""
    u = np.ascontiguousarray(v, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(v), np.uint16(0x7FC0), r).astype(np.uint16)


def from_bits(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def store(v, dt):
    return np.ascontiguousarray(v, np.float32) if dt == hip.DT_F32 else to_bits(v)


def value(a, dt):
    return a if dt == hip.DT_F32 else from_bits(a)


def formula(x, groups, gamma, beta, act, lengths):
    """(result, tolerance without the output's rounding), float64; NaN where nothing is written."""
    n, s, c = x.shape
    out, tol = np.full(x.shape, np.nan), np.zeros(x.shape)
    gamma = np.ones(c) if gamma is None else gamma.astype(np.float64)
    beta = np.zeros(c) if beta is None else beta.astype(np.float64)
    with np.errstate(all="ignore"):
        for i in range(n):
            rows = min(max(int(lengths[i]), 0), s) if lengths is not None else s
            if rows == 0:
                continue
            z = x[i, :rows].astype(np.float64).reshape(rows, groups, c // groups)
            mean = z.mean(axis=(0, 2), keepdims=True)
            rstd = 1.0 / np.sqrt(((z - mean) ** 2).mean(axis=(0, 2), keepdims=True) + EPS)
            v = ((z - mean) * rstd).reshape(rows, c) * gamma + beta
            size = np.abs(z).mean(axis=(0, 2), keepdims=True)
            t = 16 * U32 * (((np.abs(z) + np.abs(mean) + size) * rstd).reshape(rows, c) * np.abs(gamma) + np.abs(beta))
            if act == hip.ACT_RELU:
                v = np.where(v < 0, 0.0, v)
            elif act == hip.ACT_SILU:
                y = v / (1.0 + np.exp(-v))
                t = 1.1 * t + 2 * U32 * (4 + np.abs(v)) * np.abs(y)
                v = y
            out[i, :rows], tol[i, :rows] = v, t
    return out, tol


def values(rng, n, s, c, dt, offset=1.0):
    x = rng.standard_normal((n, s, c)) * (0.5 + rng.random(c)) + offset * rng.standard_normal(c)
    return value(store(x.astype(np.float32), dt), dt)      # what the type holds


class Case:
    """A call on buffers with guard values between and behind the rows."""

    def __init__(self, be, n, s, c, groups, dt, act=hip.ACT_NONE, lengths=None, affine=True, x=None, row_gap=0, image_gap=0,
                 shift=0, in_place=False, seed=0, num_cu=None, offset=1.0):
        rng = np.random.default_rng(seed)
        self.be, self.dt, self.shape, self.groups, self.act, self.lengths = be, dt, (n, s, c), groups, act, lengths
        self.x = values(rng, n, s, c, dt, offset) if x is None else x
        self.gamma = (1 + 0.3 * rng.standard_normal(c)).astype(np.float32) if affine else None
        self.beta = rng.standard_normal(c).astype(np.float32) if affine else None
        self.row, self.shift, self.in_place = c + row_gap, shift, in_place
        self.image = s * self.row + image_gap
        self.size = 4 if dt == hip.DT_F32 else 2
        self.plan = be.lib.group_norm_plan(n, s, c, groups, dt, num_cu)
        self.total = shift + (n - 1) * self.image + (s - 1) * self.row + c
        flat = np.full(self.total, 7.0, np.float32)
        self.place(flat)[...] = self.x
        self.dx = be.dev(store(flat, dt))
        self.dy = self.dx if in_place else be.dev(store(np.full(self.total, 3.0, np.float32), dt))
        self.dg, self.db = (be.dev(self.gamma), be.dev(self.beta)) if affine else (None, None)
        self.dl = be.dev(np.asarray(lengths, np.int32)) if lengths is not None else None
        self.ws = be.empty((self.plan.ws_bytes // 4,)) if self.plan.ws_bytes else None

    def place(self, flat):
        st = flat.itemsize
        return np.lib.stride_tricks.as_strided(flat[self.shift:], self.shape, (self.image * st, self.row * st, st))

    def call(self, stream=None, **kw):
        p = lambda h: None if h is None else self.be.alloc.ptr(h)  # noqa: E731
        dense = self.row == self.shape[2] and self.image == self.shape[1] * self.row
        st = (0, 0) if dense else (self.image, self.row)
        args = dict(eps=EPS, act=self.act, lengths=p(self.dl), x_strides=st, y_strides=st, workspace=p(self.ws), stream=stream)
        args.update(kw)
        self.be.lib.group_norm_forward(self.plan, p(self.dx) + self.shift * self.size, p(self.dg), p(self.db),
                                       p(self.dy) + self.shift * self.size, **args)

    def check(self):
        flat = value(self.be.host(self.dy, (self.total,)), self.dt).copy()
        got = self.place(flat).astype(np.float64)
        ref, tol = formula(self.x, self.groups, self.gamma, self.beta, self.act, self.lengths)
        n, s, c = self.shape
        for i in range(n):
            rows = s if self.lengths is None else min(max(int(self.lengths[i]), 0), s)
            r = ref[i, :rows]
            assert np.array_equal(np.isnan(r), np.isnan(got[i, :rows]))
            ok = ~np.isnan(r)
            limit = (tol[i, :rows] + UNIT[self.dt] * np.abs(r))[ok]
            worst = (np.abs(got[i, :rows] - r)[ok] - limit).max(initial=-1.0)
            assert worst <= 0, (i, worst)
            rest = got[i, rows:]                                  # rows behind the length: left as they were
            assert np.array_equal(rest, self.x[i, rows:] if self.in_place else np.full_like(rest, 3.0))
        self.place(flat)[...] = np.nan
        guard = flat[~np.isnan(flat)]
        assert np.array_equal(guard, np.full_like(guard, 7.0 if self.in_place else 3.0))


def run(be, *a, **kw):
    case = Case(be, *a, **kw)
    case.call()
    case.check()


SHAPES = [  # n, s, c, groups
    (1, 1, 1, 1), (2, 1, 8, 2), (1, 7, 16, 16), (3, 50, 64, 32), (2, 49, 24, 1), (1, 130, 75, 5), (2, 33, 210, 14),
    (1, 200, 48, 3), (1, 9, 512, 32), (1, 5, 2600, 13), (2, 3, 4104, 2), (1, 700, 8, 2), (5, 64, 12, 12), (1, 40, 260, 130),
    # more channels than a workgroup's threads take at once, groups across its tiles
    (2, 90, 4104, 2), (1, 150, 2600, 13), (1, 70, 2049, 1), (1, 130, 1030, 103), (1, 1500, 48, 4),
    # images that no workgroup's registers hold
    (3, 700, 96, 1), (2, 1100, 64, 1), (1, 2100, 256, 256), (1, 9000, 16, 1), (1, 11000, 6, 1), (1, 33000, 1, 1), (2, 4500, 32, 2),
]


@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda v: "x".join(map(str, v)))
def test_matches_the_formula(backend, shape, dt):
    run(backend, *shape, dt, act=(hip.ACT_NONE, hip.ACT_RELU, hip.ACT_SILU)[sum(shape) % 3], seed=sum(shape))


@pytest.mark.parametrize("act", [hip.ACT_NONE, hip.ACT_RELU, hip.ACT_SILU])
@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
def test_activations_without_gamma_and_beta(backend, dt, act):
    run(backend, 2, 30, 32, 4, dt, act=act, affine=False)


@pytest.mark.parametrize("num_cu", [1, 3])
@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
def test_plans_for_other_sizes_of_device(backend, dt, num_cu):
    run(backend, 3, 300, 40, 5, dt, num_cu=num_cu, act=hip.ACT_SILU)


@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(6, 37, 64, 8), (6, 37, 30, 3), (6, 400, 16, 4), (6, 700, 96, 1), (6, 1100, 64, 1), (6, 90, 2600, 2)], ids=lambda v: "x".join(map(str, v)))
def test_lengths(backend, dt, shape):
    """From none to all, one beyond either end; what lies behind a length is NaN and must not be seen."""
    s = shape[1]
    lengths = [0, 1, s, s - 1, -5, s + 9]
    x = values(np.random.default_rng(4), *shape[:3], dt)
    for i, v in enumerate(lengths):
        x[i, min(max(v, 0), s):] = np.nan
    case = Case(backend, *shape, dt, act=hip.ACT_SILU, lengths=lengths, x=x)
    case.call()
    case.check()


@pytest.mark.parametrize("row_gap,image_gap,shift", [(8, 0, 0), (8, 16, 8), (3, 5, 1), (0, 24, 0), (2, 0, 6), (1, 1, 0)])
@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in_place"])
def test_strides_alignment_and_guards(backend, dt, row_gap, image_gap, shift, in_place):
    run(backend, 3, 21, 48, 6, dt, row_gap=row_gap, image_gap=image_gap, shift=shift, in_place=in_place, act=hip.ACT_RELU)
    run(backend, 2, 600, 16, 2, dt, row_gap=row_gap, image_gap=image_gap, shift=shift, in_place=in_place)
    run(backend, 2, 700, 96, 1, dt, row_gap=row_gap, image_gap=image_gap, shift=shift, in_place=in_place, lengths=[650, 3])


@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("s", [20, 900, 5000])
def test_nan_and_infinity_stay_in_their_group(backend, dt, s):
    x = values(np.random.default_rng(8), 3, s, 32, dt)
    x[0, s // 2, 5] = np.nan
    x[1, s - 1, 17] = np.inf
    x[2, 0, 31] = -np.inf
    case = Case(backend, 3, s, 32, 4, dt, x=x, act=hip.ACT_RELU)
    case.call()
    case.check()


@pytest.mark.parametrize("s", [15, 1000, 6000])
def test_values_far_from_zero(backend, s):
    """A mean of a hundred spreads; a first position far from all others; a constant group (its variance is 0)."""
    x = values(np.random.default_rng(9), 2, s, 24, hip.DT_F32) + 100.0
    x[0, 0] = -3000.0
    x[1, :, :8] = 2.5
    case = Case(backend, 2, s, 24, 3, hip.DT_F32, x=x.astype(np.float32))
    case.call()
    case.check()


def test_all_lengths_zero(backend):
    """Nothing of x is read and nothing of y written (both images of it, in either form)."""
    for s, c, g in ((12, 16, 4), (700, 96, 1)):
        x = np.full((3, s, c), np.nan, np.float32)
        case = Case(backend, 3, s, c, g, hip.DT_F32, lengths=[0, 0, -1], x=x)
        case.call()
        case.check()


def test_nothing_to_do(backend):
    for n, s in ((0, 5), (5, 0), (0, 0)):
        p = backend.lib.group_norm_plan(n, s, 8, 2, hip.DT_F32)
        backend.lib.group_norm_forward(p, None, None, None, None)


REFUSED_PLANS = [dict(n=-1), dict(s=-1), dict(c=0), dict(groups=0), dict(groups=3), dict(groups=16), dict(dt=2), dict(num_cu=-1),
                 dict(n=2 ** 40), dict(s=2 ** 40), dict(s=2 ** 30 + 1), dict(c=2 ** 30 + 2)]


@pytest.mark.parametrize("kw", REFUSED_PLANS, ids=lambda v: "-".join(f"{a}{b}" for a, b in v.items()))
def test_refused_plans(backend, kw):
    args = dict(n=2, s=4, c=8, groups=2, dt=hip.DT_F32)
    args.update(kw)
    with pytest.raises(hip.EcoError, match="group_norm"):
        backend.lib.group_norm_plan(**args)


def test_refused_calls(backend):
    case = Case(backend, 2, 6, 8, 2, hip.DT_F32)
    lib, p = backend.lib, backend.alloc.ptr
    x, y = p(case.dx), p(case.dy)
    for kw in (dict(act=3), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x_strides=(0, 7)),
               dict(y_strides=(0, 7)), dict(y_strides=(47, 8)), dict(x_strides=(-48, 8)), dict(x_strides=(0, -8)),
               dict(x_strides=(2 ** 62, 0)), dict(x_strides=(0, 2 ** 62)), dict(y_strides=(0, 2 ** 61))):
        with pytest.raises(hip.EcoError, match="group_norm"):
            case.call(**kw)
    for a, b in ((None, y), (x, None), (x + 2, y), (x, y + 1)):
        with pytest.raises(hip.EcoError, match="group_norm"):
            lib.group_norm_forward(case.plan, a, None, None, b)
    big = lib.group_norm_plan(1, 1 << 20, 64, 4, hip.DT_F32)
    if big.ws_bytes:
        with pytest.raises(hip.EcoError, match="workspace"):
            lib.group_norm_forward(big, x, None, None, y)
    other = lib.group_norm_plan(2, 6, 8, 2, hip.DT_F32)
    other.chunks += 1
    with pytest.raises(hip.EcoError, match="plan"):
        lib.group_norm_forward(other, x, None, None, y)
    assert np.array_equal(backend.host(case.dy, (case.total,)), np.full(case.total, 3.0, np.float32))   # nothing was written


def test_refused_launches(backend):
    """More workgroups than a launch has: refused before anything is launched (no pointer is read)."""
    lib = backend.lib
    for n, s, c, groups in ((1 << 24, 40000, 8, 8), (1, 32768, 1 << 24, 1 << 24)):
        with pytest.raises(hip.EcoError, match="one launch"):
            lib.group_norm_forward(lib.group_norm_plan(n, s, c, groups, hip.DT_F32), 4, None, None, 4, workspace=8)


# ---- on the device: real sizes, streams, graphs ------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 12544, 128, 32), (3, 3136, 64, 16), (1, 196, 512, 32), (2, 1568, 256, 8), (9, 1571, 210, 14),
                                   (1, 50000, 6, 3), (700, 49, 32, 4)], ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("dt", [hip.DT_F32, hip.DT_BF16], ids=["f32", "bf16"])
def test_device_sizes(hip_backend, shape, dt):
    run(hip_backend, *shape, dt, act=hip.ACT_SILU)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(hip_backend):
    """Two images whose rows lie more than 2^32 bytes apart."""
    import torch
    be = hip_backend
    n, s, c, image = 2, 300, 64, (1 << 31) + 64
    x = torch.zeros(image + s * c, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros_like(x)
    part = torch.randn(n, s, c, device="cuda").bfloat16()
    view = torch.as_strided(x, (n, s, c), (image, c, 1))
    view.copy_(part)
    p = be.lib.group_norm_plan(n, s, c, 8, hip.DT_BF16)
    ws = torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device="cuda")
    be.lib.group_norm_forward(p, x.data_ptr(), None, None, y.data_ptr(), x_strides=(image, c), y_strides=(image, c),
                              workspace=ws.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    got = torch.as_strided(y, (n, s, c), (image, c, 1)).float().cpu().numpy()
    ref, tol = formula(part.float().cpu().numpy(), 8, None, None, hip.ACT_NONE, None)
    assert (np.abs(got - ref) <= tol + UNIT[hip.DT_BF16] * np.abs(ref)).all()
    assert int((y != 0).sum()) <= n * s * c


@pytest.mark.gpu
def test_more_images_than_one_launch_takes(hip_backend):
    """17 million images of one position, of every second image's length zero: 2^32 threads and more."""
    import torch
    n, c = (1 << 24) + 77, 8
    x = torch.randn(n, c, device="cuda").bfloat16()
    y = torch.full_like(x, 3.0)
    lengths = (torch.arange(n, device="cuda") % 2).int()
    p = hip_backend.lib.group_norm_plan(n, 1, c, 2, hip.DT_BF16)
    assert p.ws_bytes == 0
    hip_backend.lib.group_norm_forward(p, x.data_ptr(), None, None, y.data_ptr(), lengths=lengths.data_ptr(),
                                       stream=torch.cuda.current_stream().cuda_stream)
    assert bool((y[0::2] == 3.0).all())
    z = x[1::2].double().reshape(-1, 2, c // 2)
    mean = z.mean(2, keepdim=True)
    rstd = 1.0 / torch.sqrt(((z - mean) ** 2).mean(2, keepdim=True) + EPS)
    want = (z - mean) * rstd
    tol = 16 * U32 * (z.abs() + mean.abs() + z.abs().mean(2, keepdim=True)) * rstd + UNIT[hip.DT_BF16] * want.abs()
    assert bool(((y[1::2].double().reshape(-1, 2, c // 2) - want).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(8, 3136, 64, 16), (1, 196, 512, 32)], ids=lambda v: "x".join(map(str, v)))
def test_two_streams_and_graph_replays(hip_backend, shape):
    """Calls on two streams at once, each with its workspace, and a captured one replayed on new inputs: the eager bits."""
    import torch
    be = hip_backend
    n, s, c, groups = shape
    p = be.lib.group_norm_plan(n, s, c, groups, hip.DT_BF16)
    ws = [torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device="cuda") for _ in range(2)]
    xs = [torch.randn(n, s, c, device="cuda").bfloat16() for _ in range(4)]

    def call(x, y, w):
        be.lib.group_norm_forward(p, x.data_ptr(), None, None, y.data_ptr(), act=hip.ACT_SILU, workspace=w.data_ptr(),
                                  stream=torch.cuda.current_stream().cuda_stream)

    want = []
    for x in xs:
        y = torch.empty_like(x)
        call(x, y, ws[0])
        want.append(y)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.zeros_like(x) for x in xs]
    for k, x in enumerate(xs):
        with torch.cuda.stream(streams[k % 2]):
            call(x, got[k], ws[k % 2])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    held, out = torch.zeros_like(xs[0]), torch.zeros_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held, out, ws[0])
    for k in (2, 0, 3, 1, 2):
        held.copy_(xs[k])
        ws[0].fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[k])
        assert float((xs[k].float() + 1).sum()) != 0.0     # the program's own eager work between the replays
