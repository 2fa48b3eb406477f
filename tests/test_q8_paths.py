"""The 8-bit row operators on the paths that large or oddly placed rows take, and what their kernels and calls may assume."""
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "jhq_gpu_b200", "csrc")
gpu = pytest.mark.gpu
U = 2.0 ** -24                          # half a unit in the last place of float32, relative


def _norm_tol(d):
    """Of a normed row's step. A thread adds at most 32 squares in sequence, or a 1024th of a long row, and the team's
    reductions at most 10 sums more; a square's h is rounded once: the sum of squares is within (max(32, d / 1024) + 13) U,
    halved by the root. The root, the mean, eps, the two products and the largest |h w| add less than 8 U."""
    return ((max(32, -(-d // 1024)) + 13) / 2 + 8) * U


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_gen(seed), device="cuda")


def _rows(values, ld, dtype, offset=0):
    """`values` as rows `ld` apart, the first `offset` elements behind a boundary."""
    n, d = values.shape
    buf = torch.zeros(n * ld + offset + d, dtype=dtype, device="cuda")
    out = buf.as_strided((n, d), (ld, 1), offset)
    out.copy_(values)
    return out


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---- kernels that start while the one before them ends ------------------------------------------------------------

@pytest.mark.parametrize("name", ["q8_rows.cu", "q8_matmul.cu"])
def test_kernels_promise_nothing_about_what_they_read(name):
    """A kernel that starts before its predecessor's writes are done must not tell the compiler that what it reads is never
    written: loads of such memory may be moved above the wait, or go past the coherent caches."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert "before_memory();" in code
    for promise in ("__restrict__", "__restrict", ".nc.", "__ldg", "ld.const"):
        assert promise not in code, promise


def _slots_as_rows(slots):
    """An 8-bit row that reads back, in float32, as the bits of the int64s `slots` (0 .. 127): scale 2^-149, a low and a
    high word each."""
    q = torch.zeros(1, 2 * len(slots), dtype=torch.int8, device="cuda")
    q[0, ::2] = slots.to(torch.int8)
    return q, torch.tensor([2.0 ** -149], device="cuda")


@gpu
@pytest.mark.parametrize("n,groups,gdim,odd", [(3, 2, 64, 0), (300, 16, 128, 0), (20000, 2, 512, 0), (20000, 1, 1000, 0), (20001, 1, 1004, 0),
                                               (5000, 3, 333, 0), (20000, 7, 9, 0), (300, 1, 256, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reads_wait_for_values_scales_and_slots(jhq, n, groups, gdim, odd, dtype):
    """The cache is written, the slots are written, and both are read, each by the kernel right before: several rows a
    thread and one, whole and odd rows. Call by call with waits, and without."""
    d, room = groups * gdim, 120
    q = torch.zeros(room, d + odd, dtype=torch.int8, device="cuda")[:, odd:]
    scale = torch.zeros(room, groups, device="cuda")
    slots = torch.zeros(n, dtype=torch.int64, device="cuda")
    out = torch.empty(n, d, dtype=dtype, device="cuda")
    cache = jhq.Q8Rows.of(q, scale, groups=groups)
    data = [(_randn(i, room, d).to(dtype), _slots_as_rows(torch.randint(0, room, (n,), generator=_gen(50 + i), device="cuda"))) for i in range(8)]

    def chain(x, rows, wait):
        for call in (lambda: jhq.q8_write(jhq.View.of(x), cache, stream=_stream()),
                     lambda: jhq.q8_read(jhq.Q8Rows.of(*rows), jhq.View.of(slots.view(torch.float32).view(1, -1)), stream=_stream()),
                     lambda: jhq.q8_read(cache, jhq.View.of(out), slots=slots.data_ptr(), stream=_stream())):
            call()
            if wait:
                torch.cuda.synchronize()
        return out.clone()

    want = []
    for x, rows in data:
        want.append(chain(x, rows, True))
        at = rows[0][0, ::2].long()
        assert torch.equal(slots, at)
        back = (q.float().view(room, groups, gdim) * scale[:, :, None]).view(room, d).to(dtype)
        assert torch.equal(want[-1], back[at])
    for _ in range(4):
        got = [chain(x, rows, False) for x, rows in data]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("t,d,n", [(1, 999, 512), (33, 999, 130), (700, 1001, 300)])
def test_products_of_packed_rows_wait_for_them(jhq, t, d, n):
    """Rows that follow one another at odd addresses, read by the product right behind the norm that writes them, and
    behind the call that writes the weights."""
    q, scale = torch.empty(t, d, dtype=torch.int8, device="cuda"), torch.empty(t, device="cuda")
    w, ws = torch.empty(n, d, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    out = torch.empty(t, n, device="cuda")
    data = [(_randn(i, t, d) * (i + 1), _randn(90 + i, n, d)) for i in range(10)]

    def chain(x, y, wait):
        for call in (lambda: jhq.q8_rms_norm(jhq.View.of(x), jhq.Q8Rows.of(q, scale), stream=_stream()),
                     lambda: jhq.q8_write(jhq.View.of(y), jhq.Q8Rows.of(w, ws), stream=_stream()),
                     lambda: jhq.q8_matmul(jhq.Q8Rows.of(q, scale), jhq.Q8Rows.of(w, ws), jhq.View.of(out), stream=_stream())):
            call()
            if wait:
                torch.cuda.synchronize()
        return out.clone()

    want = [chain(x, y, True) for x, y in data]
    for _ in range(4):
        assert all(torch.equal(chain(x, y, False), a) for (x, y), a in zip(data, want))


# ---- operands that are not the current device's (no GPU is touched) ---------------------------------------------------

class _Elsewhere:
    """As much of a tensor as a description takes, on GPU 7; nothing is behind its address."""

    def __init__(self, rows, cols, dtype):
        self.shape, self.dtype = (rows, cols), dtype

    def stride(self):
        return self.shape[1], 1

    def data_ptr(self):
        return 4096

    def get_device(self):
        return 7

    def numel(self):
        return self.shape[0] * self.shape[1]

    def is_contiguous(self):
        return True


def _operands(jhq, view, q8):
    """Each call with every operand made by view(rows, cols) or q8(rows, dim)."""
    return [(jhq.q8_rms_norm, (view(4, 64), q8(4, 64)), {}),
            (jhq.q8_matmul, (q8(4, 64), q8(8, 64), view(4, 8)), {}),
            (jhq.q8_write, (view(4, 64), q8(9, 64)), {}),
            (jhq.q8_read, (q8(9, 64), view(4, 64)), {})]


@pytest.mark.parametrize("call", range(4))
def test_memory_elsewhere_is_refused(jhq, call):
    raw_view, raw_q8 = (lambda n, d: jhq.View(4096, n, d, d, 0)), (lambda n, d: jhq.Q8Rows(4096, 8192, n, d, d, 1))
    host_view = lambda n, d: jhq.View.of(torch.zeros(n, d))  # noqa: E731
    host_q8 = lambda n, d: jhq.Q8Rows.of(torch.zeros(n, d, dtype=torch.int8), torch.zeros(n))  # noqa: E731
    far_view = lambda n, d: jhq.View.of(_Elsewhere(n, d, torch.float32))  # noqa: E731
    far_q8 = lambda n, d: jhq.Q8Rows.of(_Elsewhere(n, d, torch.int8), _Elsewhere(n, 1, torch.float32))  # noqa: E731
    for where, v, r in (("host memory", host_view, host_q8), ("GPU 7", far_view, far_q8)):
        for view, q8 in ((v, r), (v, raw_q8), (raw_view, r)):
            f, args, kw = _operands(jhq, view, q8)[call]
            with pytest.raises(ValueError, match=where):
                f(*args, **kw)
    with pytest.raises(ValueError, match="one device"):
        jhq.Q8Rows.of(_Elsewhere(4, 64, torch.int8), torch.zeros(4))


@pytest.mark.parametrize("operand", ["weight", "residual", "residual_out", "bias"])
def test_optional_operands_elsewhere_are_refused(jhq, operand):
    x, out = jhq.View(4096, 1, 64, 64, 0), jhq.Q8Rows(4096, 8192, 1, 64, 64, 1)
    with pytest.raises(ValueError, match="host memory"):
        if operand == "bias":
            jhq.q8_matmul(out, out, jhq.View(4096, 1, 1, 1, 0), bias=jhq.View.of(torch.zeros(1, 1)))
        else:
            jhq.q8_rms_norm(x, out, **{operand: jhq.View.of(torch.zeros(1, 64))})


class _Slots(_Elsewhere):
    def __init__(self, n, dtype=torch.int64, step=1, shape=None, place=7):
        super().__init__(n, 1, dtype)
        self.shape, self._step, self._place = (n,) if shape is None else shape, step, place

    def stride(self):
        return (self._step,) * len(self.shape)

    def get_device(self):
        return self._place


@pytest.mark.parametrize("slots,msg", [
    (_Slots(4, torch.int32), "int64s are needed"), (_Slots(4, torch.float32), "int64s are needed"), (_Slots(3), "4 values"),
    (_Slots(5), "4 values"), (_Slots(4, step=2), "4 values"), (_Slots(4, shape=(2, 2)), "4 values"), (_Slots(4), "not in the memory"),
    (torch.zeros(4, dtype=torch.int64), "not in the memory")])
def test_slots_that_do_not_fit_are_refused(jhq, slots, msg):
    view, cache = jhq.View(4096, 4, 64, 64, 0), jhq.Q8Rows(4096, 8192, 9, 64, 64, 1)
    with pytest.raises(ValueError, match=msg):
        jhq.q8_write(view, cache, slots=slots)
    with pytest.raises(ValueError, match=msg):
        jhq.q8_read(cache, view, slots=slots)


@gpu
def test_slots_as_a_tensor_and_as_an_address(jhq):
    q, scale = torch.zeros(9, 64, dtype=torch.int8, device="cuda"), torch.zeros(9, device="cuda")
    cache, x = jhq.Q8Rows.of(q, scale), _randn(1, 4, 64)
    slots = torch.tensor([8, -1, 0, 3], device="cuda")
    outs = []
    for given in (slots, slots.data_ptr()):
        q.zero_()
        scale.zero_()
        jhq.q8_write(jhq.View.of(x), cache, slots=given, stream=_stream())
        out = torch.empty(4, 64, device="cuda")
        jhq.q8_read(cache, jhq.View.of(out), slots=given, stream=_stream())
        outs.append(out)
    assert torch.equal(*outs) and not outs[0][1].any() and outs[0][0].any()
    with pytest.raises(ValueError, match="4 values"):
        jhq.q8_read(cache, jhq.View.of(out), slots=slots[:3], stream=_stream())
    with pytest.raises(ValueError, match="int64s"):
        jhq.q8_write(jhq.View.of(x), cache, slots=slots.int(), stream=_stream())


# ---- a weight next to the largest float32 ------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("d", [64, 1024, 5003, 70000])
@pytest.mark.parametrize("size", [1.5, 1.9, 3e30, 1.9e-30])
def test_norm_whose_product_with_the_weight_leaves_the_range(jhq, d, size):
    """h * w is beyond float32 where h is not yet divided by its norm; the normed row is not. What is rounded to 8 bits has
    seen 6 roundings, and 1 / a, which is subnormal here, one to 2^-149: within 127 (6u + 2^-22) < 8e-5 of a step."""
    x = torch.full((3, d), size, device="cuda")
    x[:, ::3] *= -0.5
    w = torch.full((d,), 1.5e38, device="cuda")
    w[1::4] = 2.5e38
    q, scale = torch.empty(3, d, dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda")
    jhq.q8_rms_norm(jhq.View.of(x), jhq.Q8Rows.of(q, scale), weight=jhq.View.of(w), eps=0.0, stream=_stream())
    h = x.double()
    y = h / h.square().mean(1, keepdim=True).sqrt() * w.double()
    step = y.abs().amax(1, keepdim=True) / 127
    assert float(y.abs().max()) < 3.4e38                       # else the row itself is not finite
    assert torch.all((scale.double()[:, None] - step).abs() <= _norm_tol(d) * step)
    assert torch.all((q.double() * step - y).abs() <= (0.5 + 8e-5) * step)


# ---- the paths of many rows, ragged rows and rows off their boundaries -------------------------------------------------
#
# Tolerances: _norm_tol() for a step; what is rounded to 8 bits has seen at most 7 roundings, 127 * 7 U < 6e-5 of a step.

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _check_q8(q, scale, y, step_tol):
    step = y.abs().amax(-1, keepdim=True) / 127
    assert torch.all((scale.double().view(step.shape) - step).abs() <= step_tol * step + 2.0 ** -149)
    assert torch.all((q.double() * step - y).abs() <= (0.5 + 6e-5) * step + 2.0 ** -149)
    assert int(q.min()) >= -127


def _blank(rows, d, at, dtype, fill):
    """`rows` rows of d at distance at[0], at[1] elements behind a boundary, and a check that nothing beside them changed."""
    buf = torch.full((rows * at[0] + at[1],), fill, dtype=dtype, device="cuda")
    view = buf.as_strided((rows, d), (at[0], 1), at[1])

    def beside():
        gap = buf[at[1]:].view(rows, at[0])[:, d:]
        return bool((gap == fill).all()) and bool((buf[:at[1]] == fill).all())
    return view, beside


def _norm_and_check(jhq, rows, d, dtype, rtype, x_at, r_at, o_at, q_at):
    """Each *_at: (distance of rows, elements behind a boundary) of x, residual, residual_out and q."""
    x, w = _rows(_randn(1, rows, d) * 3, x_at[0], dtype, x_at[1]), (1 + 0.3 * _randn(2, d)).to(dtype)
    (q, q_beside), scale = _blank(rows, d, q_at, torch.int8, 99), torch.full((rows,), -1.0, device="cuda")
    h, kw = x.double(), {}
    if rtype:
        res = _rows(_randn(3, rows, d), r_at[0], rtype, r_at[1])
        res_out, o_beside = _blank(rows, d, o_at, rtype, 7.0)
        h = h + res.double()
        kw = dict(residual=jhq.View.of(res), residual_out=jhq.View.of(res_out))
    jhq.q8_rms_norm(jhq.View.of(x), jhq.Q8Rows.of(q, scale), weight=jhq.View.of(w), stream=_stream(), **kw)
    y = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    _check_q8(q, scale, y, _norm_tol(d))
    assert q_beside()
    if rtype:
        assert torch.equal(res_out, (x.float() + res.float()).to(rtype)) and o_beside()


def _up(n, to):
    return -(-n // to) * to


TYPES = [(BF, BF), (BF, FL), (FL, FL), (HF, None), (FL, None), (HF, HF)]
MANY = [(20001, 64), (20001, 100), (20001, 128), (20001, 130), (20001, 250), (20001, 256), (20001, 300), (20001, 500), (20001, 512), (20001, 600),
        (20001, 1003), (20001, 1024), (9001, 2003), (9001, 2048), (4001, 5001), (2001, 9001), (701, 16001), (20, 20001)]


@gpu
@pytest.mark.parametrize("rows,d", MANY)
@pytest.mark.parametrize("dtype,rtype", TYPES)
def test_norm_of_many_rows_on_boundaries(jhq, rows, d, dtype, rtype):
    ld = _up(d, 16)
    _norm_and_check(jhq, rows, d, dtype, rtype, (ld, 0), (ld, 0), (ld, 0), (ld, 0))


@gpu
@pytest.mark.parametrize("rows,d", [(20001, 100), (20001, 1003), (9001, 2003), (20001, 512), (3, 1000), (5, 4001), (300, 777), (2001, 9001)])
@pytest.mark.parametrize("dtype,rtype", TYPES)
@pytest.mark.parametrize("odd", ["out", "q", "both", "out_shifted", "q_shifted"])
def test_norm_with_outputs_off_their_boundaries(jhq, rows, d, dtype, rtype, odd):
    ld, off = _up(d, 16), (d + 1 - d % 2, 0)
    if "shifted" in odd:
        off = (ld + 16, 5)
    _norm_and_check(jhq, rows, d, dtype, rtype, (ld, 0), (ld, 0), off if odd[:3] == "out" or odd == "both" else (ld, 0),
                    off if odd[0] == "q" or odd == "both" else (ld, 0))


@gpu
@pytest.mark.parametrize("rows,d", [(20001, 7), (20001, 100), (20001, 200), (9001, 300), (9001, 500), (4001, 700), (2001, 1500), (1001, 2900), (601, 6000),
                                    (601, 9001)])
@pytest.mark.parametrize("dtype,rtype,odd", [(t, r, odd) for t, r in TYPES for odd in ("x", "residual") if odd == "x" or r])
def test_norm_of_many_rows_off_their_boundaries(jhq, rows, d, dtype, rtype, odd):
    ld = _up(d, 16)
    _norm_and_check(jhq, rows, d, dtype, rtype, (ld + 1, 1) if odd == "x" else (ld, 0), (ld, 0) if odd == "x" else (ld + 3, 1), (ld, 0), (ld, 0))


@gpu
@pytest.mark.parametrize("n,groups,gdim", [(20001, 1, 11), (20001, 1, 27), (20001, 1, 60), (20001, 1, 100), (20001, 1, 333), (20001, 1, 1003), (9001, 1, 2003),
                                           (601, 1, 9001), (9001, 16, 128), (9001, 4, 16), (9001, 4, 32), (9001, 4, 64), (9001, 3, 40), (9001, 2, 520),
                                           (9001, 5, 23), (2001, 2, 1501), (601, 2, 6001), (9001, 2, 1024)])
@pytest.mark.parametrize("dtype", [FL, HF, BF])
@pytest.mark.parametrize("odd", [False, True])
def test_cache_of_many_rows(jhq, n, groups, gdim, dtype, odd):
    d = groups * gdim
    ld, off, room = _up(d, 16) + odd, int(odd), n + 37
    x = _rows(_randn(4, n, d), ld, dtype, off)
    q = _rows(torch.full((room, d), 99, device="cuda"), ld, torch.int8, off)
    scale = torch.full((room, groups), -1.0, device="cuda")
    slots = torch.randperm(room, generator=_gen(5), device="cuda")[:n]
    slots[1], slots[n - 1] = -1, room
    cache = jhq.Q8Rows.of(q, scale, groups=groups)
    jhq.q8_write(jhq.View.of(x), cache, slots=slots, stream=_stream())
    kept = (slots >= 0) & (slots < room)
    at = slots[kept]
    _check_q8(q[at].reshape(-1, gdim), scale[at].reshape(-1), x[kept].double().reshape(-1, gdim), 2 * U)
    other = torch.ones(room, dtype=torch.bool, device="cuda")
    other[at] = False
    assert bool((q[other] == 99).all()) and bool((scale[other] == -1).all())
    for many in (n, 3):
        back = torch.randint(-1, room + 1, (many,), generator=_gen(6), device="cuda")
        out = _rows(torch.full((many, d), 5.0, device="cuda"), ld, dtype, off)
        jhq.q8_read(cache, jhq.View.of(out), slots=back, stream=_stream())
        to = back.clamp(0, room - 1)
        want = (q[to].float().view(-1, groups, gdim) * scale[to][:, :, None]).view(many, d).to(dtype)
        want[(back < 0) | (back >= room)] = 0
        assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("n,dim", [(80001, 128), (20001, 1000), (20001, 1004), (5001, 2048), (9501, 4000), (20003, 520)])
@pytest.mark.parametrize("dtype", [FL, HF, BF])
def test_reading_several_rows_a_thread(jhq, n, dim, dtype):
    """Every load width of the aligned read, at row counts that end inside a thread's rows."""
    room = 1000
    q = _rows(torch.randint(-127, 128, (room, dim), generator=_gen(7), device="cuda"), _up(dim, 16), torch.int8)
    scale = torch.rand(room, generator=_gen(8), device="cuda")
    slots = torch.randint(-1, room + 1, (n,), generator=_gen(9), device="cuda")
    out = torch.full((n, dim), 5.0, dtype=dtype, device="cuda")
    jhq.q8_read(jhq.Q8Rows.of(q, scale), jhq.View.of(out), slots=slots, stream=_stream())
    at = slots.clamp(0, room - 1)
    want = (q.float() * scale[:, None]).to(dtype)[at]
    want[(slots < 0) | (slots >= room)] = 0
    assert torch.equal(out, want)
