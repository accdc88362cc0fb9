"""The residual feed-forward block's operators at the edges of what their documentation allows: outputs that may be left out or
given, infinities and NaN, temperatures and operands far from 1, waits that run out, and Float32 products whose low parts matter.

Tolerances.  u = finfo(dtype).eps / 2 is one rounding, relative to the value; a sum of N terms in fp32 is off by at most N 2^-24 of
the sum of their absolute values.  Where a test says so, errors are bounded by their norm: N independent roundings add up like
their square root."""
import ctypes
import math

import pytest
import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODES = {F32: "F32", F16: "F16", BF16: "BF16"}


def code(dtype):
    from neurotensor_b200 import _lib
    return getattr(_lib, CODES[dtype])


def generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def randn(gen, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


# ---- norm: outputs in the place of others ----------------------------------------------------------------------------

def test_norm_outputs_that_overlap_are_refused():
    from neurotensor_b200 import _lib
    L = _lib.lib()
    a, b, c, w, s = (ctypes.c_void_p(64 * k) for k in range(1, 6))
    calls = {"y is h": lambda: L.ntb200_rms_norm(_lib.F32, a, 8, b, 8, w, c, c, s, 2, 8, 1e-6, None),
             "y is x, rows apart": lambda: L.ntb200_rms_norm(_lib.F32, a, 9, None, 0, w, a, None, s, 2, 8, 1e-6, None),
             "y is the residual, rows apart": lambda: L.ntb200_rms_norm(_lib.F32, a, 8, b, 9, w, b, None, s, 2, 8, 1e-6, None),
             "q is x": lambda: L.ntb200_rms_norm_int8(_lib.F32, a, 8, None, 0, w, a, s, None, 2, 8, 1e-6, None),
             "q is the residual": lambda: L.ntb200_rms_norm_int8(_lib.F32, a, 8, b, 8, w, b, s, None, 2, 8, 1e-6, None),
             "q is h": lambda: L.ntb200_rms_norm_int8(_lib.F32, a, 8, b, 8, w, c, s, c, 2, 8, 1e-6, None),
             "q is the quantised rows": lambda: L.ntb200_quantize_rows(_lib.F16, a, 8, a, s, 2, 8, None)}
    for what, call in calls.items():
        assert call() == _lib.ERR_INVALID_ARG, what
        assert b"in the place of" in L.ntb200_last_error_string(), what


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(5, 64), (5, 16383), (3, 40000), (2600, 4096), (9600, 264)])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_norm_in_place_of_an_input(rows, n, place):
    """y may be x or the residual itself."""
    from neurotensor_b200 import _lib, api
    gen = generator(n)
    x, r, w = randn(gen, rows, n, dtype=BF16), randn(gen, rows, n, dtype=BF16), randn(gen, n, dtype=BF16)
    results = []
    for y in (torch.empty_like(x), x if place == "x" else r):
        rstd = torch.empty(rows, device="cuda")
        _lib.check(_lib.lib().ntb200_rms_norm(_lib.BF16, x.data_ptr(), n, r.data_ptr(), n, w.data_ptr(), y.data_ptr(), None, rstd.data_ptr(), rows, n,
                                              1e-6, api._stream()))
        results.append((y, rstd))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,n", [(5, 1001), (2600, 4096), (9600, 264)])      # the last two stream
def test_norm_stream_in_place(rows, n, dtype):
    """h in the place of x or of the residual, grad_x in the place of h, grad_y or grad_h."""
    from neurotensor_b200 import _lib, api
    L, gen = _lib.lib(), generator(n)
    x, r, w, gh = randn(gen, rows, n, dtype=dtype), randn(gen, rows, n, dtype=dtype), randn(gen, n, dtype=dtype), randn(gen, rows, n, dtype=dtype)
    y, h, rstd = api.rms_norm(x, w, residual=r)
    for place in (0, 1):
        ins, out = [x.clone(), r.clone()], torch.empty_like(y)
        _lib.check(L.ntb200_rms_norm(code(dtype), ins[0].data_ptr(), n, ins[1].data_ptr(), n, w.data_ptr(), out.data_ptr(), ins[place].data_ptr(), None, rows,
                                     n, 1e-6, api._stream()))
        assert torch.equal(out, y) and torch.equal(ins[place], h) and torch.equal(ins[1 - place], (x, r)[1 - place])
    gx, gw = api.rms_norm_backward(h, w, rstd, x, grad_h=gh)
    ws = torch.empty(L.ntb200_rms_norm_backward_workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")
    for place in (0, 1, 2):
        ins, gw2 = [h.clone(), x.clone(), gh.clone()], torch.empty_like(gw)
        _lib.check(L.ntb200_rms_norm_backward(code(dtype), ins[0].data_ptr(), n, w.data_ptr(), rstd.data_ptr(), ins[1].data_ptr(), n, ins[2].data_ptr(), n,
                                              ins[place].data_ptr(), gw2.data_ptr(), ws.data_ptr(), rows, n, api._stream()))
        assert torch.equal(ins[place], gx) and torch.equal(gw2, gw)


# ---- norm: h without a residual -------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(3, 64), (37, 1999), (2, 40000), (9700, 64), (9600, 264), (2600, 4096), (700, 8192)])   # the last four stream
def test_h_without_a_residual_is_x(rows, n, dtype, int8):
    """h = x where no residual is given: a caller that passes memory for h finds x there, whatever the number of rows."""
    from neurotensor_b200 import _lib, api
    gen = generator(rows + n)
    x, w = randn(gen, rows, n, dtype=dtype), randn(gen, n, dtype=dtype)
    h = torch.full_like(x, 7.0)
    stat = torch.empty(rows, device="cuda")
    L = _lib.lib()
    if int8:
        y = torch.empty(rows, n, dtype=torch.int8, device="cuda")
        _lib.check(L.ntb200_rms_norm_int8(code(dtype), x.data_ptr(), n, None, 0, w.data_ptr(), y.data_ptr(), stat.data_ptr(), h.data_ptr(), rows, n,
                                          1e-6, api._stream()))
        want = api.rms_norm_int8(x, w)[:2]
    else:
        y = torch.empty_like(x)
        _lib.check(L.ntb200_rms_norm(code(dtype), x.data_ptr(), n, None, 0, w.data_ptr(), y.data_ptr(), h.data_ptr(), stat.data_ptr(), rows, n, 1e-6,
                                     api._stream()))
        y_, _, rstd = api.rms_norm(x, w)
        want = (y_, rstd)
    assert torch.equal(h, x)
    assert torch.equal(y, want[0]) and torch.equal(stat, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(3, 64), (37, 1999), (3, 40000), (9600, 264), (2600, 4096)])
def test_int8_row_that_is_not_finite(rows, n, dtype, bad, norm):
    """Its values are zeros and its scale is not finite, so everything that is made from it is NaN, never an infinity of a sign of its own."""
    from neurotensor_b200 import api
    gen = generator(n)
    x = randn(gen, rows, n, dtype=dtype)
    x[1, n - 1] = bad
    q, scale = api.rms_norm_int8(x, randn(gen, n, dtype=dtype))[:2] if norm else api.quantize_rows(x)
    assert not bool(q[1].any()) and not math.isfinite(float(scale[1]))
    assert bool(q[0].any()) and bool(q[2].any()) and bool(torch.isfinite(scale[0])) and bool(torch.isfinite(scale[2]))
    w = torch.ones(4, n, dtype=torch.int8, device="cuda")
    y = api.linear_int8(q[:3], scale[:3], w, torch.ones(4, device="cuda"), transpose_w=True)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2]).all())


# ---- norm: a wait that runs out --------------------------------------------------------------------------------------

def test_ring_selftest_refusals():
    from neurotensor_b200 import _lib
    L = _lib.lib()
    for args in ((48, 20, 16), (512, 20, 16), (64, 0, 16), (64, 1001, 16), (64, 20, None)):
        assert L.ntb200_selftest_ring_timeout(*args, None) == _lib.ERR_INVALID_ARG, args


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_ring_groups_leave_together(group):
    """A wait of the norm rings that runs out for some threads of a group ends the turn for all of them, and only for them."""
    from neurotensor_b200 import _lib, api
    L = _lib.lib()
    left = torch.full((512,), -1, dtype=torch.int32, device="cuda")
    _lib.check(L.ntb200_selftest_ring_timeout(group, 20, left.data_ptr(), api._stream()))
    assert L.ntb200_check_device_status(api._stream()) == _lib.ERR_TIMEOUT
    assert left.view(-1, group).tolist() == [[3 if g % 2 else 8] * group for g in range(512 // group)]
    assert L.ntb200_check_device_status(api._stream()) == _lib.OK          # reported once
    x, w = torch.ones(9600, 264, device="cuda"), torch.ones(264, device="cuda")
    assert float((api.rms_norm(x, w)[0] - 1).abs().max()) < 1e-6           # the context works on


# ---- distillation ----------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (3, 40000), (3, 131072), (500, 131072), (2, 450001)])
@pytest.mark.parametrize("rest", ["nothing", "-inf"])
def test_distill_nan_in_a_whole_piece(rows, vocab, dtype, rest):
    """NaN in half of a row, alone or among -inf, is the row's answer however the row is cut into pieces; other rows keep theirs."""
    from neurotensor_b200 import api
    gen = generator(vocab)
    s = randn(gen, rows, vocab, dtype=dtype)
    t, i = randn(gen, rows, 4), torch.randint(0, vocab // 4, (rows, 4), generator=gen, device="cuda")
    clean = api.distill_topk(s, t, i)
    s[1, vocab // 2:] = math.nan
    if rest == "-inf":
        s[1, vocab // 2 + 1:] = -math.inf
    loss, row, grad = api.distill_topk(s, t, i)
    assert math.isnan(float(loss)) and math.isnan(float(row[1])) and bool(torch.isnan(grad[1]).all())
    for r in (0, 2 if rows > 2 else 0):
        assert torch.equal(row[r], clean[1][r]) and torch.equal(grad[r], clean[2][r])


def distill64(s, t, i, T, rw):
    """(loss, row losses, gradient, the size of the gradient's two parts) in 64 bits; every entry is there."""
    lq = torch.log_softmax(s.double() / T, 1)
    lp = torch.log_softmax(t.double() / T, 1)
    p = lp.exp()
    terms = torch.where(p > 0, p * ((t.double() - t.double().amax(1, keepdim=True)) / T -
                                    ((t.double() - t.double().amax(1, keepdim=True)) / T).exp().sum(1, keepdim=True).log() - lq.gather(1, i)), torch.zeros_like(p))
    full = torch.zeros_like(lq).scatter_add_(1, i, p)
    c = T * rw.double()[:, None]
    return (T * T * terms.sum(1) * rw.double()).sum(), T * T * terms.sum(1), c * (lq.exp() - full), c * (lq.exp() + full)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [64, 40000, 131072, 450000])
@pytest.mark.parametrize("T", [1e-30, 1e-20, 1e-3, 1e6, 1e15])
def test_distill_temperatures_far_from_one(T, vocab, dtype):
    """T^2 and logits / T may leave the type's range where the loss, T^2 log V or T times a difference of logits, does not."""
    from neurotensor_b200 import api
    gen = generator(vocab)
    s, t = randn(gen, 5, vocab, scale=3.0, dtype=dtype), randn(gen, 5, 6, scale=3.0)
    i = torch.stack([torch.randperm(vocab, generator=gen, device="cuda")[:6] for _ in range(5)])
    rw = torch.tensor([0.5, 0.25, 1.0, 0.125, 0.0625], device="cuda")
    loss, row, grad = api.distill_topk(s, t, i, temperature=T, row_weight=rw)
    loss64, row64, grad64, size = distill64(s, t, i, T, rw)
    # exponents up to 2^6 matter: their fp32 rounding is 2^-18 of each probability; sums of vocab terms add their own
    e = 2.0 ** -17 + 2.0 ** -24 * min(vocab, 4096)
    scale = T * T * (1 + math.log(vocab + 1)) + 2 * T * float(s.float().abs().max() + t.abs().max())
    assert bool(((row.double() - row64).abs() <= e * scale).all()), (row, row64)
    assert abs(float(loss) - float(loss64)) <= e * scale * 2
    u = torch.finfo(dtype).eps / 2
    assert bool(((grad.double() - grad64).abs() <= u * (1 + 2.0 ** -7) * grad64.abs() + e * size + 2.0 ** -126).all())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [64, 40000, 131072, 450000])
@pytest.mark.parametrize("T", [0.25, 0.5])
def test_distill_teacher_names_a_column_of_the_lowest_value(T, vocab):
    """The row's loss, T p times the lowest Float32, is finite although that logit / T is not."""
    from neurotensor_b200 import api
    gen = generator(vocab)
    s = randn(gen, 2, vocab)
    i = torch.tensor([[1, vocab - 2, 7], [3, 4, 5]], device="cuda")
    s[0, vocab - 2] = torch.finfo(F32).min
    t = torch.zeros(2, 3, device="cuda")
    loss, row, grad = api.distill_topk(s, t, i, temperature=T)
    want = -T / 3 * torch.finfo(F32).min
    assert abs(float(row[0]) - want) <= 2.0 ** -20 * want and abs(float(loss) - want / 2) <= 2.0 ** -20 * want
    assert bool(torch.isfinite(grad).all())


# ---- linear in Float32 -----------------------------------------------------------------------------------------------

def infinite_pattern(x, w):
    """x @ w in 64 bits; where a row of x or a column of w holds infinities or NaN, from its products one by one."""
    y = torch.nan_to_num(x, 0, 0, 0).double() @ torch.nan_to_num(w, 0, 0, 0).double()
    for r in (~torch.isfinite(x)).any(1).nonzero().flatten().tolist():
        y[r] = (x[r].double()[:, None] * w.double()).sum(0)
    for c in (~torch.isfinite(w)).any(0).nonzero().flatten().tolist():
        y[:, c] = (x.double() * w[:, c].double()).sum(1)
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("m,k,n", [(5, 40, 33), (100, 24, 33), (200, 257, 300), (300, 2048, 513), (2600, 300, 4104)])
def test_float32_infinities(m, k, n, transpose):
    """Infinite and NaN operands give what fp32 products and sums give, on every route that a size may take."""
    from neurotensor_b200 import api
    gen = generator(m + k)
    x, w = randn(gen, m, k), randn(gen, k, n)
    w = torch.where(w.abs() < 2.0 ** -10, torch.ones_like(w), w)      # far from the low parts' end
    x = torch.where(x.abs() < 2.0 ** -10, torch.ones_like(x), x)
    x[0, 3], x[1, k - 1], x[2, 0], x[2, 9], x[3, 5], x[3, 6], x[4, 11] = math.inf, -math.inf, math.inf, math.inf, math.inf, -math.inf, math.nan
    w[3, 7] = 0.0                                                      # inf times 0
    w[3, 1], w[8, 2] = math.inf, -math.inf                             # one of them meets x[0, 3]
    y = api.linear_act(x, w.t().contiguous() if transpose else w, transpose_w=transpose)
    want = infinite_pattern(x, w)
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(y), kind(want)), kind.__name__
    fine = torch.isfinite(want)
    size = torch.nan_to_num(x, 0, 0, 0).double().abs() @ torch.nan_to_num(w, 0, 0, 0).double().abs()
    assert bool(((y.double() - want).abs()[fine] <= ((k + 4) * 2.0 ** -23 + 3 * 2.0 ** -22) * size[fine]).all())
    # a gradient that overflowed: columns of gx's terms are infinite
    gy = randn(gen, m, n)
    gy = torch.where(gy.abs() < 2.0 ** -10, torch.ones_like(gy), gy)
    gy[0, 0] = math.inf
    clean = torch.nan_to_num(w, 1.0, 1.0, 1.0)
    gx, gw, gb = api.linear_act_backward(torch.nan_to_num(x, 1.0, 1.0, 1.0), clean.t().contiguous() if transpose else clean, None, gy, transpose_w=transpose)
    assert torch.equal(gx[0].double(), math.inf * clean[:, 0].double()) and bool(torch.isfinite(gx[1:]).all())
    gw = gw.t() if transpose else gw
    assert torch.equal(gw[:, 0].double(), math.inf * torch.nan_to_num(x, 1.0, 1.0, 1.0)[0].double()) and bool(torch.isfinite(gw[:, 1:]).all())
    assert math.isinf(float(gb[0])) and bool(torch.isfinite(gb[1:]).all())


def f16_parts(x, dim):
    """The two Float16 parts (in fp32) of a matrix whose rows along `dim` are scaled so that their largest value lies in [2^14, 2^15)."""
    scale = 2.0 ** (14 - torch.floor(torch.log2(x.abs().amax(dim, keepdim=True))))
    v = x * scale
    hi = v.half().float()
    return hi / scale, (v - hi).half().float() / scale


# Error of a Float32 product as three Float16 products, by its norm, relative to the result's.  A partial sum takes 24 adds (8 steps of
# 16 along K, three products each), each cut off after 24 bits, by half a step of 2^-23 on average, while it grows to its size, so
# that an add meets 2/3 of it on average: 24 * 2^-24 * 2/3 = 2^-20.  The parts (2^-23 a value), lo.lo and the fp32 adds of the
# partial sums stay below 2^-22 together, errors of independent terms being summed by their squares.
THREE_PRODUCTS = 2.0 ** -20 + 2.0 ** -22


def relative_norm(got, want):
    return float((got.double() - want).norm() / want.norm())


def test_float32_bound_sees_a_lost_low_part():
    """Without the low part of either operand, or of an eighth of its terms, the product misses that bound by far."""
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(64, 1024, generator=gen), torch.randn(1024, 64, generator=gen)
    want = x.double() @ w.double()
    (xh, xl), (wh, wl) = ([p.double() for p in f16_parts(v, d)] for v, d in ((x, 1), (w, 0)))
    assert relative_norm(xh @ wh + xh @ wl + xl @ wh, want) < THREE_PRODUCTS / 4
    assert relative_norm(xh @ wh + xh @ wl, want) > 50 * THREE_PRODUCTS
    assert relative_norm(xh @ wh + xl @ wh, want) > 50 * THREE_PRODUCTS
    xl[:, :128] = 0
    assert relative_norm(xh @ wh + xh @ wl + xl @ wh, want) > 20 * THREE_PRODUCTS


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("m,k,n", [(100, 100, 130), (200, 257, 300), (300, 640, 513), (128, 4096, 2048), (256, 4096, 512), (590, 832, 1792),
                                   (45, 2048, 448), (64, 2048, 2048), (7, 4095, 33),                                # few rows
                                   (2600, 600, 4104), (2600, 130, 4103), (2601, 1000, 4104), (1100, 2048, 3001)])   # CTA pairs, several partial sums
def test_float32_products(m, k, n, transpose):
    """Forward, pre-activation and both gradients against 64 bits by the norm of the error."""
    from neurotensor_b200 import api
    gen = generator(m + k + n)
    x, w, gy = randn(gen, m, k), randn(gen, k, n), randn(gen, m, n)
    wt = w.t().contiguous() if transpose else w
    want = x.double() @ w.double()
    assert relative_norm(api.linear_act(x, wt, transpose_w=transpose), want) < THREE_PRODUCTS
    _, pre = api.linear_act(x, wt, None, "silu", transpose_w=transpose, want_pre=True)
    assert relative_norm(pre, want) < THREE_PRODUCTS
    gx, gw, gb = api.linear_act_backward(x, wt, None, gy, transpose_w=transpose)
    assert relative_norm(gx, gy.double() @ w.double().t()) < THREE_PRODUCTS
    assert relative_norm(gw.t() if transpose else gw, x.double().t() @ gy.double()) < THREE_PRODUCTS
    assert relative_norm(gb, gy.double().sum(0)) < THREE_PRODUCTS


@pytest.mark.gpu
@pytest.mark.parametrize("up", [13, 20, 26])
@pytest.mark.parametrize("m,k,n", [(200, 1024, 300), (2600, 600, 4104)])
def test_float32_values_far_below_their_rows_largest(m, k, n, up):
    """One value of 2^up in each row of x meets weights of 0: what the others lose is at most 2^-39 of it each."""
    from neurotensor_b200 import api
    gen = generator(up)
    x, w = randn(gen, m, k).clamp(-8, 8), randn(gen, k, n)
    x[:, 5], w[5] = 2.0 ** up, 0.0
    want = x.double() @ w.double()
    lost = 2.0 ** (up - 39) * w.double().abs().sum(0, keepdim=True).expand_as(want)
    assert float((api.linear_act(x, w).double() - want).norm()) <= THREE_PRODUCTS * float(want.norm()) + float(lost.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16, torch.int8])
@pytest.mark.parametrize("m,k,n", [(2600, 72, 4104), (2600, 72, 4103), (300, 512, 1024), (16, 4096, 4096)])
def test_linear_in_place_of_its_residual(m, k, n, dtype, pre):
    """y in the residual's place, on the epilogues of CTA pairs (residuals by TMA or by rows), single tiles and K slices."""
    from neurotensor_b200 import _lib, api
    gen = generator(m + n)
    out = BF16 if dtype == torch.int8 else dtype
    bias, r = randn(gen, n, dtype=out), randn(gen, m, n, dtype=out)
    if dtype == torch.int8:
        x = torch.randint(-127, 128, (m, k), generator=gen, device="cuda", dtype=dtype)
        w = torch.randint(-127, 128, (k, n), generator=gen, device="cuda", dtype=dtype)
        s, v = torch.rand(m, generator=gen, device="cuda") * 0.01, torch.rand(n, generator=gen, device="cuda") * 0.01
    else:
        x, w = randn(gen, m, k, dtype=dtype), randn(gen, k, n, scale=k ** -0.5, dtype=dtype)
    results = []
    for y in (torch.empty_like(r), r):
        d, _, keep, stream = api._linear_desc("linear", x, w, bias, "gelu", r, False, out)
        if dtype == torch.int8:
            d.x_scale, d.w_scale = s.data_ptr(), v.data_ptr()
        z = torch.empty_like(r)
        if pre:
            d.pre, d.pre_row_stride = z.data_ptr(), n
        api._run_linear(d, y, stream)
        results.append((y.clone(), z))
    assert torch.equal(results[0][0], results[1][0]) and (not pre or torch.equal(results[0][1], results[1][1]))
