"""The 8-bit row operators (jhq_q8_*) against their formulas in 64 bits, and their refusals.

Tolerances, with u = 2^-24 (half a unit in the last place of float32, relative):
- h = x + r and g = h * w are one rounding each, so a = max |g| is within 2u of its value, and
  g * (127 * (1 / a)), with three more roundings, within 7u of its, at most 127 * 7u < 6e-5 of a step: a written
  value is within 0.5 + 6e-5 steps of the formula's.
- the step of the norm: the sum of d squares, each within 3u (two roundings of h, one of the square), in
  partial sums of at most d / 32 + 16 terms in sequence, so within (d / 32 + 19) u, halved by the root; the root,
  the mean, eps and the two products add less than 8u.
- a product: the conversion of the exact sum, two products and one sum: 4u of |sum| + |bias|; then the rounding
  to the output's type (2^-8 bfloat16, 2^-11 float16, none for float32).
"""
import ctypes as C

import pytest
import torch

U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_gen(seed), device="cuda")


def _strided(v, ld, dtype, offset=0):
    """v as rows `ld` apart, the first `offset` elements behind a boundary."""
    n, d = v.shape
    buf = torch.zeros(n * ld + offset + d, dtype=dtype, device="cuda")
    out = buf.as_strided((n, d), (ld, 1), offset)
    out.copy_(v)
    return out


def _q8(seed, rows, dim, ld=None, offset=0, lo=-127):
    q = torch.randint(lo, 128, (rows, dim), generator=_gen(seed), device="cuda")
    return _strided(q, ld or dim, torch.int8, offset), torch.rand(rows, generator=_gen(seed + 1), device="cuda") + 0.01


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _check_rows(q, scale, y, step_tol):
    """q * scale against the formula's y (float64), and the step itself."""
    top = y.abs().amax(-1, keepdim=True)
    step = top / 127
    got = scale.double().view(step.shape)
    assert torch.all((got - step).abs() <= step_tol * step + 2.0 ** -149)
    err = (q.double() * step - y).abs()
    assert torch.all(err <= (0.5 + 6e-5) * step + 2.0 ** -149), float((err / step.clamp(min=1e-300)).max())
    assert int(q.abs().max()) <= 127


def _norm_tol(d):
    return ((d / 32 + 19) / 2 + 8) * U


NORM_SHAPES = [  # rows, dim, padding of x, offset of x in elements
    (1, 1, 0, 0), (3, 2, 1, 0), (1, 7, 0, 1), (5, 31, 0, 3), (33, 64, 0, 0), (300, 100, 0, 0), (257, 128, 0, 0),
    (64, 129, 7, 5), (1, 1000, 0, 0), (130, 1024, 0, 0), (7, 1025, 0, 1), (513, 2048, 8, 0), (1, 4096, 0, 0),
    (40, 4096, 0, 0), (9, 5003, 0, 0), (2, 8192, 16, 8), (150, 8200, 0, 0), (1, 16384, 0, 0), (3, 40001, 0, 0),
    (2, 70000, 0, 0), (1, 131072, 0, 0)]


def _norm_case(jhq, rows, d, pad, off, dtype, rtype, weight, inplace=False, eps=1e-6, x=None, r=None, w=None):
    x = _randn(1, rows, d) * 3 if x is None else x
    x = _strided(x, d + pad, dtype, off)
    ld_q = (d + 15) // 16 * 16 if off == 0 else d + 1
    q = _strided(torch.full((rows, d), 99, device="cuda"), ld_q, torch.int8, off)
    scale = torch.full((rows,), -1.0, device="cuda")
    w = (1 + 0.3 * _randn(2, d)).to(dtype if weight == "same" else torch.float32) if w is None and weight else w
    res = res_out = None
    if rtype:
        res = _strided(_randn(3, rows, d) if r is None else r, d + 2 * pad, rtype, off)
        before = res.clone()
        res_out = res if inplace else torch.full((rows, d), 7.0, dtype=rtype, device="cuda")
    jhq.q8_rms_norm(jhq.View.of(x), jhq.Q8Rows.of(q, scale), weight=None if w is None else jhq.View.of(w),
                    residual=None if res is None else jhq.View.of(res),
                    residual_out=None if res is None else jhq.View.of(res_out), eps=eps, stream=_stream())
    h = x.double()
    if rtype:
        h = h + before.double()
        assert torch.allclose(res_out, (x.float() + before.float()).to(rtype), rtol=0, atol=0, equal_nan=True)
    y = h / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return q, scale, y if w is None else y * w.double()


@gpu
@pytest.mark.parametrize("rows,d,pad,off", NORM_SHAPES)
@pytest.mark.parametrize("dtype,rtype,weight", [("bf16", "bf16", "same"), ("f16", "f32", "f32"), ("f32", "f32", None),
                                                ("bf16", None, "f32"), ("f16", "f16", "same"), ("bf16", "f32", "same")])
def test_rms_norm(jhq, rows, d, pad, off, dtype, rtype, weight):
    q, scale, y = _norm_case(jhq, rows, d, pad, off, DT[dtype], DT[rtype] if rtype else None, weight)
    _check_rows(q, scale, y, _norm_tol(d))


@gpu
@pytest.mark.parametrize("d", [96, 1024, 4096, 40001])
def test_rms_norm_residual_in_place(jhq, d):
    q, scale, y = _norm_case(jhq, 37, d, 0, 0, torch.bfloat16, torch.bfloat16, "same", inplace=True)
    _check_rows(q, scale, y, _norm_tol(d))


@gpu
@pytest.mark.parametrize("d", [8, 100, 1024, 4096, 8200, 70000])
def test_rms_norm_zero_and_nonfinite_rows(jhq, d):
    x = _randn(5, 8, d)
    x[0] = 0
    x[2, d // 2] = float("inf")
    x[4, 0] = float("nan")
    x[5, d - 1] = float("-inf")
    q, scale, y = _norm_case(jhq, 8, d, 0, 0, torch.float32, torch.float32, "f32", x=x, r=torch.zeros(8, d, device="cuda"))
    assert float(scale[0]) == 0 and not q[0].any()
    for i in (2, 4, 5):
        assert torch.isnan(scale[i]) and not q[i].any()
    for i in (1, 3, 6, 7):
        _check_rows(q[i:i + 1], scale[i:i + 1], y[i:i + 1], _norm_tol(d))


@gpu
@pytest.mark.parametrize("d", [64, 1024, 5003, 70000])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("size", [1e-42, 1e-30, 1e-21, 1e18, 1e30, 2e37])
def test_rms_norm_at_the_ends_of_the_range(jhq, d, eps, size):
    """Squares that leave float32's range; the weight takes part of a product out of it too."""
    x = _randn(6, 4, d).clamp(-4, 4) * size
    w = torch.ones(d, device="cuda")
    w[: d // 2] = 8.0 if size > 1 else 0.25
    q, scale, y = _norm_case(jhq, 4, d, 0, 0, torch.float32, None, None, eps=eps, x=x, w=w)
    if size >= 1e-37 and float(y.abs().max()) > 1e-30:         # else the inputs or the steps are subnormal
        _check_rows(q, scale, y, _norm_tol(d))
    else:
        step = y.abs().amax(1) / 127
        assert torch.all((scale.double() - step).abs() <= 1e-3 * step + 2.0 ** -149)


@gpu
@pytest.mark.parametrize("d", [100, 4096])
def test_rms_norm_weight_of_zeros_and_one_value(jhq, d):
    w = torch.zeros(d, device="cuda")
    q, scale, _ = _norm_case(jhq, 3, d, 0, 0, torch.bfloat16, None, None, w=w)
    assert not q.any() and not scale.any()
    w[d - 1] = -2
    q, scale, y = _norm_case(jhq, 3, d, 0, 0, torch.bfloat16, None, None, w=w)
    _check_rows(q, scale, y, _norm_tol(d))
    assert torch.equal(q[:, d - 1].abs(), torch.full((3,), 127, dtype=torch.int8, device="cuda"))


# ---- the product ------------------------------------------------------------------------------------------

MM_SHAPES = [  # tokens, channels, depth
    (1, 1, 1), (1, 5, 3), (2, 129, 16), (1, 128, 4096), (3, 1000, 999), (8, 256, 128), (16, 300, 144), (17, 640, 4097),
    (32, 127, 8192), (33, 2048, 1024), (64, 1024, 512), (65, 513, 1000), (100, 104, 104), (127, 1024, 256),
    (128, 128, 128), (129, 257, 4096), (200, 1024, 1024), (255, 255, 255), (256, 1024, 4096), (257, 129, 130),
    (500, 77, 1001), (512, 512, 16), (1000, 999, 1001), (1024, 4096, 128), (2049, 1025, 640), (5000, 333, 4096),
    (1, 20000, 256), (40, 10007, 48), (9000, 16, 64), (1, 64, 131071), (300, 300, 131071)]


def _mm_check(jhq, t, n, k, dtype, bias, ldx=None, ldw=None, offx=0, offw=0, ldo=None, offo=0, lo=-127):
    qx, sx = _q8(11, t, k, ldx, offx, lo)
    qw, sw = _q8(13, n, k, ldw, offw, lo)
    b = _randn(15, n) * 50 if bias else None
    out = _strided(torch.full((t, n), 3.0, device="cuda"), ldo or n, dtype, offo)
    jhq.q8_matmul(jhq.Q8Rows.of(qx, sx), jhq.Q8Rows.of(qw, sw), jhq.View.of(out),
                  bias=jhq.View.of(b) if bias else None, stream=_stream())
    y = (qx.double() @ qw.double().T) * sx.double()[:, None] * sw.double()
    mag = y.abs()
    if bias:
        mag, y = mag + b.double().abs(), y + b.double()
    tol = 4.1 * U * mag
    if dtype != torch.float32:
        tol = tol + HALF_ULP[dtype] * (y.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    got = out.double()
    if dtype == torch.float16:                 # what rounds to an infinity is one
        over = y.abs() > 65504
        assert torch.all(torch.isinf(got[y.abs() > 65600]))
        got, y = torch.where(over, 0, got), torch.where(over, 0, y)
    assert torch.all((got - y).abs() <= tol), float(((got - y).abs() / tol.clamp(min=1e-300)).max())
    jhq.q8_check_status()
    return out


@gpu
@pytest.mark.parametrize("t,n,k", MM_SHAPES)
@pytest.mark.parametrize("dtype,bias", [("f32", True), ("bf16", False), ("f16", True)])
def test_matmul(jhq, t, n, k, dtype, bias):
    """Rows that begin on 16-byte boundaries, rows that follow one another, and rows at odd addresses."""
    pad = (k + 15) // 16 * 16
    _mm_check(jhq, t, n, k, DT[dtype], bias, ldx=pad, ldw=pad)
    if k % 16:
        _mm_check(jhq, t, n, k, DT[dtype], bias)
    _mm_check(jhq, t, n, k, DT[dtype], bias, ldx=k + 3, ldw=pad, offx=5)
    _mm_check(jhq, t, n, k, DT[dtype], bias, ldx=pad, ldw=k + 16, offw=1, ldo=n + 5, offo=3)


@gpu
@pytest.mark.parametrize("t,n,k", [(1, 128, 1024), (40, 300, 131071), (300, 520, 999), (1030, 515, 1024)])
def test_matmul_sums_are_exact(jhq, t, n, k):
    """Scales of one, no bias: float32 outputs are the integer sums, rounded once. -128 counts too."""
    for fill in (None, -128):
        qx, qw = _q8(21, t, k, (k + 15) // 16 * 16, lo=-128)[0], _q8(23, n, k, (k + 15) // 16 * 16, lo=-128)[0]
        if fill is not None:
            qx.fill_(fill)
            qw.fill_(fill)
        one = torch.ones(max(t, n), device="cuda")
        out = torch.empty(t, n, device="cuda")
        jhq.q8_matmul(jhq.Q8Rows.of(qx, one[:t]), jhq.Q8Rows.of(qw, one[:n]), jhq.View.of(out), stream=_stream())
        assert torch.equal(out, (qx.double() @ qw.double().T).float())


@gpu
def test_matmul_repeats_bit_for_bit(jhq):
    for t, n, k in ((1, 4096, 4096), (48, 1000, 8192), (700, 900, 2048)):
        a = _mm_check(jhq, t, n, k, torch.float32, True)
        b = _mm_check(jhq, t, n, k, torch.float32, True)
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("t", [1, 70, 400])
def test_matmul_nonfinite_scales_stay_in_their_rows(jhq, t):
    qx, sx = _q8(31, t, 256)
    qw, sw = _q8(33, 200, 256)
    sx[0] = float("nan")
    sw[7] = float("inf")
    out = torch.empty(t, 200, device="cuda")
    jhq.q8_matmul(jhq.Q8Rows.of(qx, sx), jhq.Q8Rows.of(qw, sw), jhq.View.of(out), stream=_stream())
    assert torch.isnan(out[0]).all()
    fine = torch.ones(200, dtype=torch.bool, device="cuda")
    fine[7] = False
    assert torch.isfinite(out[1:, fine]).all() and not torch.isfinite(out[1:, 7]).any()


@gpu
@pytest.mark.parametrize("t", [1, 300])
def test_matmul_writes_only_its_output(jhq, t):
    n, k, ldo = 131, 160, 140
    qx, sx = _q8(41, t, k)
    qw, sw = _q8(43, n, k)
    buf = torch.full((t + 2, ldo), 5.0, device="cuda")
    jhq.q8_matmul(jhq.Q8Rows.of(qx, sx), jhq.Q8Rows.of(qw, sw), jhq.View.of(buf[1:t + 1, 4:4 + n]), stream=_stream())
    assert bool((buf[0] == 5).all() and (buf[t + 1] == 5).all() and (buf[:, :4] == 5).all() and (buf[:, 4 + n:] == 5).all())


@gpu
@pytest.mark.parametrize("t", [3, 130])
def test_matmul_far_rows(jhq, t):
    """Row offsets beyond 2^31 bytes in every operand."""
    n, k = 65, 96
    far = (2 ** 31 // (t - 1) + 4096) // 16 * 16
    big = torch.empty(far * t + 64, dtype=torch.int8, device="cuda")
    qx = big.as_strided((t, k), (far, 1))
    qx.copy_(torch.randint(-127, 128, (t, k), generator=_gen(5), device="cuda"))
    wfar = 2 ** 31 // (n - 1) // 16 * 16 + 64
    wbig = torch.empty(wfar * n + 64, dtype=torch.int8, device="cuda")
    qw = wbig.as_strided((n, k), (wfar, 1))
    qw.copy_(torch.randint(-127, 128, (n, k), generator=_gen(6), device="cuda"))
    obig = torch.empty(far * t + 64, dtype=torch.bfloat16, device="cuda")
    out = obig.as_strided((t, n), (far, 1))
    one = torch.ones(max(t, n), device="cuda")
    jhq.q8_matmul(jhq.Q8Rows.of(qx, one[:t]), jhq.Q8Rows.of(qw, one[:n]), jhq.View.of(out), stream=_stream())
    assert torch.equal(out, (qx.double() @ qw.double().T).bfloat16())


# ---- the cache ----------------------------------------------------------------------------------------------

CACHE_SHAPES = [  # new rows, groups, dim of a group
    (1, 1, 1), (5, 3, 1), (3, 1, 5), (1, 16, 128), (70, 8, 64), (33, 5, 23), (2, 1, 1024), (100, 2, 100), (9, 1, 4096),
    (4, 3, 1001), (300, 32, 16), (17, 4, 80), (2, 1, 33000), (1000, 1, 128), (40, 2, 256), (6, 7, 520), (3, 2, 9000)]


@gpu
@pytest.mark.parametrize("n,groups,gdim", CACHE_SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("odd", [0, 3])
def test_cache_write_and_read(jhq, n, groups, gdim, dtype, odd):
    d, room = groups * gdim, 2 * n + 5
    x = _strided(_randn(51, n, d) * 2, d + odd, DT[dtype], odd)
    x[n // 2, : gdim] = 0
    ld = (d + 15) // 16 * 16 if not odd else d + odd
    q, _ = _q8(53, room, d, ld, odd)
    scale = torch.rand(room, groups, generator=_gen(54), device="cuda")
    q0, s0 = q.clone(), scale.clone()
    slots = torch.randperm(room, generator=_gen(55), device="cuda")[:n]
    if n > 2:
        slots[1], slots[n - 1] = -1, room                      # padding, and one behind the cache
    rows = jhq.Q8Rows.of(q, scale, groups=groups)
    jhq.q8_write(jhq.View.of(x), rows, slots=slots.data_ptr(), stream=_stream())
    kept = (slots >= 0) & (slots < room)
    _check_rows(q[slots[kept]].reshape(-1, gdim), scale[slots[kept]].reshape(-1), x[kept].double().reshape(-1, gdim), 2 * U)
    other = torch.ones(room, dtype=torch.bool, device="cuda")
    other[slots[kept]] = False
    assert torch.equal(q[other], q0[other]) and torch.equal(scale[other], s0[other])

    back = torch.randint(0, room, (3 * n + 1,), generator=_gen(56), device="cuda")
    back[0] = -1
    back[-1] = room + 7
    out = _strided(torch.full((len(back), d), 5.0, device="cuda"), d + odd, DT[dtype], odd)
    jhq.q8_read(rows, jhq.View.of(out), slots=back.data_ptr(), stream=_stream())
    at = back.clamp(0, room - 1)
    want = (q[at].float().view(-1, groups, gdim) * scale[at][:, :, None]).view(-1, d).to(DT[dtype])
    want[0], want[-1] = 0, 0
    assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("groups,gdim", [(1, 384), (4, 96), (1, 12000)])
def test_cache_without_slots_and_nonfinite_groups(jhq, groups, gdim):
    n, d = 6, groups * gdim
    x = _randn(61, n, d)
    x[1, gdim // 2], x[3, gdim - 1] = float("nan"), float("inf")
    q, scale = torch.empty(n, d, dtype=torch.int8, device="cuda"), torch.empty(n, groups, device="cuda")
    rows = jhq.Q8Rows.of(q, scale, groups=groups)
    jhq.q8_write(jhq.View.of(x), rows, stream=_stream())
    for i in (1, 3):
        assert torch.isnan(scale[i, 0]) and not q[i, :gdim].any()
        if groups > 1:
            assert torch.isfinite(scale[i, 1:]).all()
    fine = [0, 2, 4, 5]
    _check_rows(q[fine].reshape(-1, gdim), scale[fine].reshape(-1), x[fine].double().reshape(-1, gdim), 2 * U)
    out = torch.empty(n, d, device="cuda")
    jhq.q8_read(rows, jhq.View.of(out), stream=_stream())
    want = (q.float().view(n, groups, gdim) * scale[:, :, None]).view(n, d)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())


@gpu
@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-30, 1e30, 1e38])
def test_cache_write_at_the_ends_of_the_range(jhq, size):
    x = _randn(63, 5, 512).clamp(-3, 3) * size
    q, scale = torch.empty(5, 512, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
    jhq.q8_write(jhq.View.of(x), jhq.Q8Rows.of(q, scale), stream=_stream())
    top = x.double().abs().amax(1, keepdim=True)
    assert torch.all((q.double() - x.double() * 127 / top).abs() <= 0.5 + 6e-5)
    assert torch.all((scale.double() - top[:, 0] / 127).abs() <= 2 * U * top[:, 0] / 127 + 2.0 ** -149)


@gpu
def test_cache_of_more_than_4_gib(jhq):
    d, room = 1024, 2 ** 32 // 1024 + 3000
    q, scale = torch.empty(room, d, dtype=torch.int8, device="cuda"), torch.zeros(room, 2, device="cuda")
    slots = torch.tensor([room - 1, 2 ** 31 // d + 1, 2 ** 32 // d + 2, 0], device="cuda")
    x = _randn(65, 4, d)
    rows = jhq.Q8Rows.of(q, scale, groups=2)
    jhq.q8_write(jhq.View.of(x), rows, slots=slots.data_ptr(), stream=_stream())
    out = torch.empty(4, d, device="cuda")
    jhq.q8_read(rows, jhq.View.of(out), slots=slots.data_ptr(), stream=_stream())
    step = x.abs().view(4, 2, -1).amax(2) / 127
    assert torch.all((out - x).view(4, 2, -1).abs() <= 0.501 * step[:, :, None])
    assert torch.equal(scale[slots], step)


# ---- how they are called ------------------------------------------------------------------------------------

@gpu
def test_no_rows(jhq):
    e8, e32 = torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda")
    empty = torch.empty(0, 64, device="cuda")
    q, s = _q8(71, 3, 64)
    out = torch.full((3, 64), 2.0, device="cuda")
    jhq.q8_rms_norm(jhq.View.of(empty), jhq.Q8Rows.of(e8, e32))
    jhq.q8_matmul(jhq.Q8Rows.of(e8, e32), jhq.Q8Rows.of(q, s), jhq.View.of(torch.empty(0, 3, device="cuda")))
    jhq.q8_matmul(jhq.Q8Rows.of(q, s), jhq.Q8Rows.of(e8, e32), jhq.View.of(torch.empty(3, 0, device="cuda")))
    jhq.q8_write(jhq.View.of(empty), jhq.Q8Rows.of(q, s))
    jhq.q8_write(jhq.View.of(out), jhq.Q8Rows.of(e8, e32), slots=torch.zeros(3, dtype=torch.int64, device="cuda").data_ptr())
    jhq.q8_read(jhq.Q8Rows.of(q, s), jhq.View.of(empty))
    assert bool((out == 2).all())
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    jhq.q8_read(jhq.Q8Rows.of(e8, e32), jhq.View.of(out), slots=slots.data_ptr())
    assert not out.any()                                       # every slot is outside an empty cache


@gpu
def test_on_a_side_stream_and_in_a_graph(jhq):
    t, d, n = 24, 512, 256
    x, (w, ws) = _randn(81, t, d).bfloat16(), _q8(83, n, d)
    q, scale = torch.empty(t, d, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda")
    out = torch.empty(t, n, device="cuda")

    def head():
        rows = jhq.Q8Rows.of(q, scale)
        jhq.q8_rms_norm(jhq.View.of(x), rows, stream=_stream())
        jhq.q8_matmul(rows, jhq.Q8Rows.of(w, ws), jhq.View.of(out), stream=_stream())

    head()
    want = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        head()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        head()
    x.copy_(_randn(85, t, d))
    g.replay()
    replayed = out.clone()
    out.zero_()
    head()
    assert torch.equal(replayed, out) and not torch.equal(replayed, want)


@gpu
@pytest.mark.parametrize("t,d,n", [(1, 1024, 512), (40, 4096, 1000), (700, 640, 300), (3000, 512, 1024), (33, 999, 130)])
def test_calls_wait_for_one_another(jhq, t, d, n):
    """Kernels start while the one before them ends: a chain over shared buffers gives what it gives call by call."""
    w, ws = _q8(87, n, d, (d + 15) // 16 * 16)
    q, scale = _q8(88, t, d, (d + 15) // 16 * 16)
    h, back, kept = torch.empty(t, n, device="cuda"), torch.empty(t, n, device="cuda"), _q8(89, t, n)

    def chain(x, wait):
        rows, cache = jhq.Q8Rows.of(q, scale), jhq.Q8Rows.of(*kept)
        for call in (lambda: jhq.q8_rms_norm(jhq.View.of(x), rows, stream=_stream()),
                     lambda: jhq.q8_matmul(rows, jhq.Q8Rows.of(w, ws), jhq.View.of(h), stream=_stream()),
                     lambda: jhq.q8_write(jhq.View.of(h), cache, stream=_stream()),
                     lambda: jhq.q8_read(cache, jhq.View.of(back), stream=_stream())):
            call()
            if wait:
                torch.cuda.synchronize()
        return back.clone()

    xs = [_randn(200 + i, t, d) * (i + 1) for i in range(12)]
    want = [chain(x, True) for x in xs]
    for _ in range(4):
        got = [chain(x, False) for x in xs]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("t,n,k,packed", [(1, 1024, 8192, False), (100, 300, 4096, False), (40, 300, 999, True),
                                          (700, 900, 640, False), (5000, 2000, 2048, False)])
def test_waits_that_give_up_are_reported(jhq, monkeypatch, t, n, k, packed):
    """With no cycles to wait (JHQ_TEST_TC_WAIT_CYCLES, read at the launch) every wait gives up: the kernel ends by
    itself, the status says so once, and the next call is whole again."""
    monkeypatch.setenv("JHQ_TEST_TC_WAIT_CYCLES", "0")
    qx, sx = _q8(95, t, k, k if packed else None)
    qw, sw = _q8(96, n, k, k if packed else None)
    out = torch.zeros(t, n, device="cuda")
    jhq.q8_matmul(jhq.Q8Rows.of(qx, sx), jhq.Q8Rows.of(qw, sw), jhq.View.of(out), stream=_stream())
    torch.cuda.synchronize()
    with pytest.raises(jhq.JHQError) as e:
        jhq.q8_check_status()
    assert e.value.code == jhq.JHQ_ETIMEDOUT
    jhq.q8_check_status()
    monkeypatch.delenv("JHQ_TEST_TC_WAIT_CYCLES")
    _mm_check(jhq, t, n, k, torch.float32, False)


@gpu
def test_launches_are_counted(jhq):
    x = _randn(91, 4, 64)
    q, s = torch.empty(4, 64, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    n = jhq.kernel_launches()
    jhq.q8_write(jhq.View.of(x), jhq.Q8Rows.of(q, s))
    jhq.q8_matmul(jhq.Q8Rows.of(q, s), jhq.Q8Rows.of(q, s), jhq.View.of(torch.empty(4, 4, device="cuda")))
    assert jhq.kernel_launches() >= n + 2


@gpu
def test_example_finds_the_queries_items():
    """A query's embedding has a cosine of about 0.99 with its item's and one of at most about 6 / sqrt(128) = 0.53 with any
    of 5000 others: the first result is its item unless a kernel is wrong."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "q8_embedding_search.py")
    spec = importlib.util.spec_from_file_location("q8_embedding_search", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(n=5000, nq=200) >= 0.99


# ---- refusals (no GPU is touched) -----------------------------------------------------------------------------

def _v(jhq, rows=4, cols=64, ld=None, kind=0, data=4096):
    return jhq.View(data, rows, cols, cols if ld is None else ld, kind)


def _r(jhq, rows=4, dim=64, ld=None, groups=1, q=4096, scale=8192):
    return jhq.Q8Rows(q, scale, rows, dim, dim if ld is None else ld, groups)


NORM_REFUSED = [
    (dict(x=dict(kind=3)), "unknown type"), (dict(x=dict(kind=-1)), "unknown type"), (dict(x=dict(data=None)), "null data"),
    (dict(x=dict(ld=63)), "smaller than a row"), (dict(x=dict(data=4098)), "aligned"), (dict(x=dict(rows=-1)), "rows"),
    (dict(x=dict(cols=0, ld=0)), "cols"), (dict(out=dict(rows=3)), "rows and cols"), (dict(out=dict(dim=32)), "rows and cols"),
    (dict(out=dict(groups=2)), "one group"), (dict(out=dict(groups=3)), "divide"), (dict(out=dict(groups=0)), "divide"),
    (dict(out=dict(q=None)), "null buffer"), (dict(out=dict(scale=None)), "null buffer"), (dict(out=dict(scale=8194)), "aligned"),
    (dict(out=dict(ld=10)), "smaller than a row"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(weight=dict(rows=2)), "1 x cols"), (dict(weight=dict(rows=1, cols=32)), "1 x cols"),
    (dict(weight=dict(rows=1, kind=2)), "x's type or float32"), (dict(residual=dict(rows=3)), "rows and cols"),
    (dict(residual=dict(kind=1)), "x's type or float32"), (dict(residual_out=dict(cols=63)), "rows and cols"),
    (dict(x=dict(kind=2), residual=dict(kind=2), residual_out=dict(kind=0)), "one type")]


@pytest.mark.parametrize("change,msg", NORM_REFUSED)
def test_rms_norm_refuses(jhq, change, msg):
    kw = {k: _v(jhq, **change[k]) for k in ("weight", "residual", "residual_out") if k in change}
    with pytest.raises(ValueError, match=msg):
        jhq.q8_rms_norm(_v(jhq, **change.get("x", {})), _r(jhq, **change.get("out", {})), eps=change.get("eps", 1e-6), **kw)


@pytest.mark.parametrize("change,msg", [
    (dict(x=dict(dim=32)), "one length"), (dict(x=dict(dim=131072), w=dict(dim=131072)), "131071"),
    (dict(x=dict(groups=2)), "one group"), (dict(w=dict(groups=2)), "one group"), (dict(out=dict(rows=3)), "x's rows by w's rows"),
    (dict(out=dict(cols=9)), "x's rows by w's rows"), (dict(out=dict(kind=7)), "unknown type"), (dict(out=dict(ld=4)), "smaller"),
    (dict(bias=dict(rows=1, cols=7)), "bias"), (dict(bias=dict(rows=2, cols=8)), "bias"), (dict(bias=dict(rows=1, cols=8, kind=1)), "bias"),
    (dict(x=dict(q=None)), "null buffer"), (dict(w=dict(scale=None)), "null buffer"), (dict(out=dict(data=None)), "null data"),
    (dict(x=dict(dim=0)), "dim")])
def test_matmul_refuses(jhq, change, msg):
    x, w = _r(jhq, **change.get("x", {})), _r(jhq, **dict(dict(rows=8), **change.get("w", {})))
    out = _v(jhq, **dict(dict(rows=4, cols=8), **change.get("out", {})))
    with pytest.raises(ValueError, match=msg):
        jhq.q8_matmul(x, w, out, bias=_v(jhq, **change["bias"]) if "bias" in change else None)


@pytest.mark.parametrize("change,msg", [
    (dict(v=dict(cols=32)), "as long as the cache"), (dict(v=dict(rows=9)), "more rows"), (dict(slots=4100), "aligned"),
    (dict(r=dict(groups=5)), "divide"), (dict(v=dict(kind=5)), "unknown type"), (dict(r=dict(q=None)), "null buffer")])
def test_cache_refuses(jhq, change, msg):
    v, r = _v(jhq, **change.get("v", {})), _r(jhq, **dict(dict(rows=8), **change.get("r", {})))
    with pytest.raises(ValueError, match=msg):
        jhq.q8_write(v, r, slots=change.get("slots"))
    with pytest.raises(ValueError, match=msg):
        jhq.q8_read(r, v, slots=change.get("slots"))


def test_null_arguments_and_tensors_that_do_not_fit(jhq):
    L = jhq.load_library()
    assert L.jhq_q8_rms_norm(None, None, None, 1e-6, None, None, None) == jhq.JHQ_EINVAL
    assert L.jhq_q8_matmul(None, None, None, None, None) == jhq.JHQ_EINVAL
    assert L.jhq_q8_write(None, None, None, None) == jhq.JHQ_EINVAL
    assert L.jhq_q8_read(None, None, None, None) == jhq.JHQ_EINVAL
    assert b"null" in L.jhq_last_error()
    t = torch.zeros(4, 6)
    assert (jhq.View.of(t[:, :3]).ld, jhq.View.of(t[0]).rows) == (6, 1)
    for bad, msg in ((t.T, "follow one another"), (t.double(), "float32"), (t.view(2, 2, 6), "2-D")):
        with pytest.raises(ValueError, match=msg):
            jhq.View.of(bad)
    with pytest.raises(ValueError, match="int8"):
        jhq.Q8Rows.of(t, t[:, 0])
    with pytest.raises(ValueError, match="packed scales"):
        jhq.Q8Rows.of(t.to(torch.int8), torch.zeros(3))
    with pytest.raises(C.ArgumentError):
        jhq.q8_read(jhq.View.of(t), jhq.View.of(t))
