"""Norm with residual, linear with activation and residual, Int8 linear with scales and the distillation loss, against
plain 64-bit restatements.

Tolerances.  u = finfo(dtype).eps / 2 is one rounding, relative to the value; a value that fp32 arithmetic reaches through
sums of N terms is off by at most N 2^-24 of the sum of their absolute values (2^-23 on the tensor cores, whose adds
truncate).  Each test adds up the roundings that its operator's definition contains."""
import ctypes
import math

import pytest
import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half a step below the normal range: what a rounding to a subnormal may lose (fp32 results are flushed to nothing less)."""
    return {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}[dtype]


def randn(gen, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def same_but_order(got, want):
    """Equal but for the order of the fp32 sums behind them, which may follow the layout: at most one step of the type."""
    return got.shape == want.shape and bool(((got.double() - want.double()).abs() <= torch.finfo(got.dtype).eps * (8 if got.dtype == F32 else 1) *
                                             want.double().abs().clamp(min=1e-30)).all())


def generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def within(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d values off, worst by %.3g of its tolerance" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).max()))


def act64(z, act):
    """(value, slope) in 64 bits."""
    if act == "relu":
        return z.clamp(min=0), (z >= 0).double()
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        g = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return z * g, g + z * g * (1 - g) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    return z, torch.ones_like(z)


# ---- refusals, on the CPU -------------------------------------------------------------------------------------------

def test_norm_refusals():
    from neurotensor_b200 import _lib, api
    L = _lib.lib()
    one = ctypes.c_void_p(16)
    for call in (lambda: L.ntb200_rms_norm(_lib.I8, one, 8, None, 0, one, one, None, None, 1, 8, 1e-6, None),
                 lambda: L.ntb200_quantize_rows(_lib.F64, one, 8, one, one, 1, 8, None)):
        assert call() == _lib.ERR_UNSUPPORTED
    for call in (lambda: L.ntb200_rms_norm(_lib.F32, one, 8, None, 0, one, one, None, None, -1, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 8, None, 0, one, one, None, None, 1, 0, 1e-6, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 8, None, 0, None, one, None, None, 1, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 8, None, 0, one, one, None, None, 1, 8, -1.0, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 8, None, 0, one, one, None, None, 1, 8, float("nan"), None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 7, None, 0, one, one, None, None, 2, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 8, one, 7, one, one, None, None, 2, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, one, 9, None, 0, one, ctypes.c_void_p(64), one, None, 2, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm(_lib.F32, ctypes.c_void_p(32), 8, one, 9, one, ctypes.c_void_p(64), one, None, 2, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm_backward(_lib.F32, ctypes.c_void_p(32), 8, one, one, one, 9, None, 0, one, None, None, 2, 8, None),
                 lambda: L.ntb200_rms_norm_int8(_lib.F32, one, 8, None, 0, one, one, None, None, 2, 8, 1e-6, None),
                 lambda: L.ntb200_rms_norm_backward(_lib.F32, one, 8, one, one, one, 8, None, 0, one, one, None, 2, 8, None),
                 lambda: L.ntb200_rms_norm_backward(_lib.F32, one, 8, one, one, one, 8, one, 7, one, None, None, 2, 8, None)):
        assert call() == _lib.ERR_INVALID_ARG
    assert L.ntb200_rms_norm(_lib.F32, None, 8, None, 0, None, None, None, None, 0, 8, 1e-6, None) == _lib.OK   # no rows
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        api.rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="weight"):
        api.rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="residual"):
        api.rms_norm(x, torch.ones(8), residual=torch.zeros(2, 8, dtype=F16))
    with pytest.raises(ValueError, match="Float32"):
        api.rms_norm_int8(x.int(), torch.ones(8))
    with pytest.raises(ValueError, match="rstd"):
        api.rms_norm_backward(x, torch.ones(8), torch.ones(3), x)


def test_linear_refusals():
    from neurotensor_b200 import _lib, api
    L = _lib.lib()

    def call(**kw):
        d = _lib.LinearDesc()
        base = dict(dtype=_lib.F16, out_dtype=_lib.F16, activation=0, m=4, n=8, k=8, x=16, x_row_stride=8, x_col_stride=1, w=16,
                    w_row_stride=8, w_col_stride=1, y=48, y_row_stride=8)
        base.update(kw)
        for name, v in base.items():
            setattr(d, name, v)
        return L.ntb200_linear_act(ctypes.byref(d), None, 0, None)

    assert L.ntb200_linear_act(None, None, 0, None) == _lib.ERR_INVALID_ARG
    assert call(dtype=_lib.F64, out_dtype=_lib.F64) == _lib.ERR_UNSUPPORTED
    for kw in (dict(out_dtype=_lib.F32), dict(activation=9), dict(m=-1), dict(x_row_stride=-8), dict(y_row_stride=7), dict(y=None),
               dict(x=None), dict(dtype=_lib.I8), dict(dtype=_lib.I8, x_scale=16, w_scale=16, k=131072, x_row_stride=131072),
               dict(x_scale=16, w_scale=16), dict(pre=48, pre_row_stride=8), dict(residual=32, residual_row_stride=4), dict(y=16), dict(pre=16, pre_row_stride=8),
               dict(residual=48, residual_row_stride=16), dict(dtype=_lib.I8, out_dtype=_lib.I8, x_scale=16, w_scale=16)):
        assert call(**kw) == _lib.ERR_INVALID_ARG, kw
    assert call(m=0) == _lib.OK and call(n=0) == _lib.OK

    def back(**kw):
        d = _lib.LinearBackwardDesc()
        base = dict(dtype=_lib.F16, activation=1, m=4, n=8, k=8, x=16, x_row_stride=8, x_col_stride=1, w=16, w_row_stride=8,
                    w_col_stride=1, pre=16, pre_row_stride=8, grad_out=16, grad_out_row_stride=8, grad_x=48, grad_w=64, grad_bias=80)
        base.update(kw)
        for name, v in base.items():
            setattr(d, name, v)
        return L.ntb200_linear_act_backward(ctypes.byref(d), None, 0, None)

    assert back(dtype=_lib.I8) == _lib.ERR_UNSUPPORTED
    for kw in (dict(pre=None), dict(grad_out=None), dict(w=None), dict(x=None), dict(activation=-1), dict(grad_out_row_stride=3),
               dict(k=0), dict(grad_x=16), dict(grad_w=16), dict(grad_bias=16)):
        assert back(**kw) == _lib.ERR_INVALID_ARG, kw

    x, w = torch.zeros(3, 4), torch.zeros(4, 5)
    for bad in (lambda: api.linear_act(x, w), lambda: api.linear_act(x, torch.zeros(5, 5)), lambda: api.linear_act(x, w.half()),
                lambda: api.linear_act(x, w, bias=torch.zeros(4)), lambda: api.linear_act(x, w, residual=torch.zeros(3, 4)),
                lambda: api.linear_act(x.int(), w.int()), lambda: api.linear_int8(x, torch.zeros(3), w, torch.zeros(5)),
                lambda: api.linear_act_backward(x, w, None, torch.zeros(3, 5), "relu"),
                lambda: api.linear_act_backward(x, w, torch.zeros(3, 5), torch.zeros(3, 4), "relu")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="activation"):
        api._activation("tanh")


def test_distill_refusals():
    from neurotensor_b200 import _lib, api
    L = _lib.lib()

    def call(dtype=_lib.F32, s_rs=8, tdt=_lib.F32, idt=_lib.I32, grad=64, g_rs=8, rows=2, vocab=8, top=3, temp=1.0, logits=16, loss=16):
        return L.ntb200_distill_topk(dtype, logits, s_rs, tdt, 16, idt, 16, None, grad, g_rs, 16, loss, rows, vocab, top, temp, None)

    assert call(dtype=_lib.I32) == _lib.ERR_UNSUPPORTED and call(tdt=_lib.F64) == _lib.ERR_UNSUPPORTED and call(idt=_lib.I16) == _lib.ERR_UNSUPPORTED
    for kw in (dict(rows=-1), dict(vocab=0), dict(top=0), dict(top=1025), dict(temp=0.0), dict(temp=-1.0), dict(temp=1e-31), dict(temp=float("inf")),
               dict(temp=float("nan")), dict(s_rs=7), dict(g_rs=7), dict(logits=None), dict(loss=None), dict(grad=16, g_rs=16)):
        assert call(**kw) == _lib.ERR_INVALID_ARG, kw
    s, t, i = torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)
    for bad in (lambda: api.distill_topk(s, t, i), lambda: api.distill_topk(s, t, i.short()), lambda: api.distill_topk(s, t[:1], i),
                lambda: api.distill_topk(s, t, i, temperature=0.0), lambda: api.distill_topk(s, t, i, row_weight=torch.ones(3)),
                lambda: api.distill_topk(s, torch.zeros(2, 1025), torch.zeros(2, 1025, dtype=torch.int32)),
                lambda: api.distill_topk(s.int(), t, i)):
        with pytest.raises(ValueError):
            bad()


# ---- norm -----------------------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (3, 5), (7, 64), (130, 200), (1, 4096), (37, 1999), (5, 8192), (3, 16384), (2, 16383), (2, 40000), (300, 33), (1000, 256),
               (9700, 64), (9600, 264), (2600, 2048), (1300, 4104), (700, 8192), (650, 16384),     # enough rows to stream
               (1000, 1001), (260, 14054)]


def norm_inputs(rows, n, dtype, residual, seed=0):
    gen = generator(seed + rows * 131 + n)
    x = randn(gen, rows, n, dtype=dtype)
    r = randn(gen, rows, n, scale=3.0, dtype=dtype) if residual else None
    w = (1 + randn(gen, n, scale=0.3)).to(dtype)
    return gen, x, r, w


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", NORM_SHAPES)
def test_norm(rows, n, dtype, residual):
    from neurotensor_b200 import api
    _, x, r, w = norm_inputs(rows, n, dtype, residual)
    y, h, rstd = api.rms_norm(x, w, eps=1e-5, residual=r)
    h64 = x.double() + (r.double() if residual else 0)
    rstd64 = (h64.pow(2).mean(1) + 1e-5).rsqrt()
    e = n * 2.0 ** -24 / 2 + 8 * 2.0 ** -24        # the sum of squares under a root, and a handful of operations
    within(rstd, rstd64, e * rstd64, "rstd")
    y64 = h64 * rstd64[:, None] * w.double()
    slack = 2.0 ** -24 * (x.double().abs() + (r.double().abs() if residual else 0)) * rstd64[:, None] * w.double().abs()   # h itself in fp32
    within(y, y64, (half_step(dtype) + e) * y64.abs() + slack + smallest(dtype), "y")
    if residual:
        within(h, h64, half_step(dtype) * h64.abs() * (1 + 2.0 ** -10) + 2.0 ** -24 * (x.double().abs() + r.double().abs()) + smallest(dtype), "h")
    else:
        assert h is x


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", NORM_SHAPES)
def test_norm_int8(rows, n, dtype, residual):
    """q follows its definition in fp32 bit for bit, so every value equals the plain restatement's."""
    from neurotensor_b200 import api
    _, x, r, w = norm_inputs(rows, n, dtype, residual, 1)
    q, scale, h = api.rms_norm_int8(x, w, eps=1e-5, residual=r)
    hf = x.float() + r.float() if residual else x.float()
    u = hf * w.float()
    top = u.abs().amax(1)
    want = torch.clamp(torch.round(u * (torch.full_like(top, 127.0) / top)[:, None]), -127, 127)
    assert torch.equal(q.float(), want)
    h64 = hf.double()
    s64 = top.double() * (h64.pow(2).mean(1) + 1e-5).rsqrt() / 127
    within(scale, s64, (n * 2.0 ** -25 + 8 * 2.0 ** -24) * s64, "scale")
    if residual:
        assert torch.equal(h, hf.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(1, 1), (9, 77), (64, 1024), (3, 40000)])
def test_quantize_rows(rows, n, dtype):
    from neurotensor_b200 import api
    x = randn(generator(rows + n), rows, n, dtype=dtype)
    x[0] = 0                                                 # a row of zeros: scale 0, values 0
    q, scale = api.quantize_rows(x)
    assert float(scale[0]) == 0 and not bool(q[0].any())
    top = x.float().abs().amax(1)
    inv = torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))
    assert torch.equal(q.float(), torch.clamp(torch.round(x.float() * inv[:, None]), -127, 127))
    assert torch.equal(scale, top / torch.full_like(top, 127.0))     # a true division: by a number, torch multiplies by its reciprocal
    # half a step of q, and the three fp32 roundings of x * (127 / A) on a value of up to 127: 127 * 3 * 2^-24 steps
    step = scale.double()[:, None] * (0.5 + 127 * 3 * 2.0 ** -24)
    assert bool(((q.double() * scale.double()[:, None] - x.double()).abs() <= step).all())


@pytest.mark.gpu
def test_quantize_rows_extremes():
    from neurotensor_b200 import api
    tiny = torch.tensor([[1e-39, -5e-40, 0.0, 2.5e-40]], device="cuda")
    q, scale = api.quantize_rows(tiny)                       # 127 / max would overflow
    assert q.tolist() == [[127, -64, 0, 32]] or q.tolist() == [[127, -63, 0, 32]]
    x = torch.ones(3, 8, device="cuda")
    x[0, 3], x[1, 5] = float("nan"), float("inf")
    q, scale = api.quantize_rows(x)
    assert math.isnan(float(scale[0])) and math.isinf(float(scale[1])) and float(scale[2]) == float(torch.tensor(1.0) / 127)
    w = torch.ones(4, 8, dtype=torch.int8, device="cuda")
    y = api.linear_int8(q, scale, w, torch.ones(4, device="cuda"), transpose_w=True, dtype=F32)
    assert not bool(torch.isfinite(y[:2]).any()) and bool(torch.isfinite(y[2]).all())


def norm_backward64(h, w, gy, gh, eps):
    """Gradient of sum(gy . y + gh . h) with respect to h, and to w, by differentiation in 64 bits."""
    h = h.double().requires_grad_()
    w = w.double().requires_grad_()
    y = h * (h.pow(2).mean(1, keepdim=True) + eps).rsqrt() * w
    total = (gy.double() * y).sum() + ((gh.double() * h).sum() if gh is not None else 0)
    return torch.autograd.grad(total, (h, w))


@pytest.mark.gpu
@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", NORM_SHAPES)
def test_norm_backward(rows, n, dtype, stream):
    from neurotensor_b200 import api
    gen, h, _, w = norm_inputs(rows, n, dtype, False, 2)
    gy = randn(gen, rows, n, dtype=dtype)
    gh = randn(gen, rows, n, dtype=dtype) if stream else None
    _, _, rstd = api.rms_norm(h, w, eps=1e-5)
    gx, gw = api.rms_norm_backward(h, w, rstd, gy, grad_h=gh)
    gx64, gw64 = norm_backward64(h, w, gy, gh, 1e-5)
    inv = rstd.double()[:, None]
    g, xhat = (gy.double() * w.double()).abs(), h.double().abs() * inv
    e = (n + 16) * 2.0 ** -24
    tol = half_step(dtype) * gx64.abs() + e * (inv * (g + xhat * (g * xhat).mean(1, keepdim=True))) + smallest(dtype)
    if stream:
        tol = tol + 2.0 ** -23 * gh.double().abs()
    within(gx, gx64, tol, "gx")
    within(gw, gw64, half_step(dtype) * gw64.abs() + (rows + n + 16) * 2.0 ** -24 * (gy.double().abs() * xhat).sum(0) + smallest(dtype), "gw")
    again = api.rms_norm_backward(h, w, rstd, gy, grad_h=gh)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)          # a fixed order
    only = api.rms_norm_backward(h, w, rstd, gy, grad_h=gh, want_weight=False)
    assert only[1] is None and torch.equal(only[0], gx)


@pytest.mark.gpu
def test_norm_layouts():
    """Leading dims, padded rows, transposed and expanded inputs, views that do not start on 16 bytes, no rows at all."""
    from neurotensor_b200 import api
    gen = generator(5)
    big = randn(gen, 6, 7, 100, dtype=BF16)
    w = randn(gen, 64, dtype=BF16)
    for x in (big[..., :64], big[..., 1:65], big[:, 0, :64], big.permute(1, 0, 2)[..., 3:67], big[0, 0, :64],
              randn(gen, 64, 9, dtype=BF16).t(), w[None, :].expand(5, 64)):
        y, h, rstd = api.rms_norm(x, w, residual=x)
        ref = api.rms_norm(x.contiguous(), w, residual=x.contiguous())
        assert same_but_order(y, ref[0]) and torch.equal(h, ref[1]) and same_but_order(rstd, ref[2]) and y.shape == x.shape
        gx, gw = api.rms_norm_backward(x, w, rstd, x, grad_h=x)
        ref = api.rms_norm_backward(x.contiguous(), w, rstd, x.contiguous(), grad_h=x.contiguous())
        # gx = gh + rstd (g - xhat c) may cancel: a step of its largest part
        assert float((gx.double() - ref[0].double()).abs().max()) <= 2.0 ** -7 * float(x.abs().max()) and gx.shape == x.shape
        assert float((gw.double() - ref[1].double()).abs().max()) <= 2.0 ** -7 * float(ref[1].abs().max())
    y, _, _ = api.rms_norm(big[:0, :, :64], w)
    assert y.shape == (0, 7, 64)
    gx, gw = api.rms_norm_backward(big[:0, 0, :64], w, torch.zeros(0, device="cuda"), big[:0, 0, :64])
    assert gx.shape == (0, 64) and not bool(gw.any())
    # the rows before and behind are left as they were
    out = torch.full((4, 64), 7.0, dtype=BF16, device="cuda")
    from neurotensor_b200 import _lib
    x = randn(gen, 2, 64, dtype=BF16)
    _lib.check(_lib.lib().ntb200_rms_norm(_lib.BF16, x.data_ptr(), 64, None, 0, w.data_ptr(), out[1].data_ptr(), None, None, 2, 64,
                                          1e-6, api._stream()))
    assert bool((out[0] == 7).all()) and bool((out[3] == 7).all()) and torch.equal(out[1:3], api.rms_norm(x, w)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 4096, 16383, 40000])
def test_norm_in_place_of_the_stream(n):
    """h may take the residual's place, and grad_x the place of an incoming gradient."""
    from neurotensor_b200 import _lib, api
    gen = generator(n)
    x, r, w = randn(gen, 5, n, dtype=BF16), randn(gen, 5, n, dtype=BF16), randn(gen, n, dtype=BF16)
    y, h, rstd = api.rms_norm(x, w, residual=r)
    y2, r2 = torch.empty_like(y), r.clone()
    _lib.check(_lib.lib().ntb200_rms_norm(_lib.BF16, x.data_ptr(), n, r2.data_ptr(), n, w.data_ptr(), y2.data_ptr(), r2.data_ptr(), None, 5, n,
                                          1e-6, api._stream()))
    assert torch.equal(y2, y) and torch.equal(r2, h)
    gx, gw = api.rms_norm_backward(h, w, rstd, x, grad_h=r)
    g2, gw2 = x.clone(), torch.empty_like(gw)
    ws = torch.empty(_lib.lib().ntb200_rms_norm_backward_workspace_bytes(5, n), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().ntb200_rms_norm_backward(_lib.BF16, h.data_ptr(), n, w.data_ptr(), rstd.data_ptr(), g2.data_ptr(), n, r.data_ptr(), n,
                                                   g2.data_ptr(), gw2.data_ptr(), ws.data_ptr(), 5, n, api._stream()))
    assert torch.equal(g2, gx) and torch.equal(gw2, gw)


# ---- linear ---------------------------------------------------------------------------------------------------------

LINEAR_SHAPES = [(1, 1, 1), (1, 64, 8), (3, 7, 5), (5, 40, 33), (16, 512, 256), (33, 100, 130), (128, 4096, 2048), (129, 72, 200),
                 (200, 257, 300), (300, 640, 513), (1, 4096, 4096), (64, 4096, 4096), (256, 4096, 512), (1100, 136, 1032),
                 (2600, 72, 4104), (2600, 72, 4103)]      # several tiles per CTA pair


def linear_tolerance(x64, w64, k, dtype, y64, extra=0.0):
    """Roundings of y = act(z) + r: the fp32 sum of z through a slope of at most 1.13, the fp32 activation (a few 2^-21 of
    its value for 16-bit results, 2^-22 for Float32), the residual's add, one rounding."""
    z_err = (k + 4) * 2.0 ** -23 * (x64.abs() @ w64.abs()) + extra
    if dtype == F32:      # three products of parts that carry 21 bits or more: 3 2^-22 of each product besides
        z_err = z_err + 3 * 2.0 ** -22 * (x64.abs() @ w64.abs())
    return 1.13 * z_err, 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", LINEAR_SHAPES)
def test_linear_act(m, k, n, dtype, act):
    from neurotensor_b200 import api
    gen = generator(m + 7 * k + 31 * n)
    x, w = randn(gen, m, k, dtype=dtype), randn(gen, k, n, scale=1.5 / math.sqrt(k), dtype=dtype)
    b = randn(gen, n, scale=0.5, dtype=dtype) if (m + n) % 3 else None
    r = randn(gen, m, n, dtype=dtype) if (m + k) % 2 or act == "gelu" else None
    z64 = x.double() @ w.double() + (b.double() if b is not None else 0)
    v64, slope = act64(z64, act)
    y64 = v64 + (r.double() if r is not None else 0)
    zt, rel = linear_tolerance(x.double(), w.double(), k, dtype, y64)
    if b is not None:
        zt = zt + 2.0 ** -23 * b.double().abs()
    tol = half_step(dtype) * y64.abs() * (1 + 2.0 ** -9) + zt + rel * (v64.abs() + z64.abs() * 2.0 ** -3) + 2.0 ** -23 * y64.abs() + smallest(dtype)
    for transpose in (False, True):
        wt = w.t().contiguous() if transpose else w
        y, pre = api.linear_act(x, wt, b, act, residual=r, transpose_w=transpose, want_pre=True)
        within(y, y64, tol, "y")
        within(pre, z64, half_step(dtype) * z64.abs() * (1 + 2.0 ** -9) + zt + smallest(dtype), "pre")
        assert torch.equal(api.linear_act(x, wt, b, act, residual=r, transpose_w=transpose), y)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (3, 7, 5), (33, 100, 130), (130, 257, 300), (300, 640, 513), (1, 2048, 2048), (700, 512, 1024)])
def test_linear_act_backward(m, k, n, dtype, act):
    from neurotensor_b200 import api
    gen = generator(m + 5 * k + 3 * n)
    x, w = randn(gen, m, k, dtype=dtype), randn(gen, k, n, scale=1.0 / math.sqrt(k), dtype=dtype)
    pre, gy = randn(gen, m, n, scale=1.5, dtype=dtype), randn(gen, m, n, dtype=dtype)
    _, slope = act64(pre.double(), act)
    gz = gy.double() * slope
    u = half_step(dtype)
    gz_err = (u if dtype != F32 and act != "none" else 0) * gz.abs() * (1 + 2.0 ** -9) + gy.double().abs() * 2.0 ** -19 + smallest(dtype)
    mult = 2.0 ** -23 + (3 * 2.0 ** -22 if dtype == F32 else 0)
    for transpose in (False, True):
        wt = w.t().contiguous() if transpose else w
        gx, gw, gb = api.linear_act_backward(x, wt, pre, gy, act, transpose_w=transpose)
        gx64, gw64, gb64 = gz @ w.double().t(), x.double().t() @ gz, gz.sum(0)
        a = gz.abs() + gz_err
        within(gx, gx64, u * gx64.abs() * (1 + 2.0 ** -9) + gz_err @ w.double().abs().t() + (n * 2.0 ** -23 + mult) * (a @ w.double().abs().t()) + smallest(dtype), "gx")
        gw = gw.t() if transpose else gw
        within(gw, gw64, u * gw64.abs() * (1 + 2.0 ** -9) + x.double().abs().t() @ gz_err + (m * 2.0 ** -23 + mult) * (x.double().abs().t() @ a) + smallest(dtype), "gw")
        within(gb, gb64, u * gb64.abs() * (1 + 2.0 ** -9) + ((m + 8) * 2.0 ** -24 + 2.0 ** -19) * gy.double().abs().sum(0) * 1.2 + smallest(dtype), "gb")
        only = api.linear_act_backward(x, wt, pre, gy, act, transpose_w=transpose, want_x=False, want_bias=False)
        assert only[0] is None and only[2] is None and torch.equal(only[1].t() if transpose else only[1], gw)
        assert torch.equal(api.linear_act_backward(x, wt, pre, gy, act, transpose_w=transpose)[2], gb)     # a fixed order


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_linear_gradients_are_differences(act):
    """The gradients against central differences of the forward pass (Float32): step e = 2^-6, third derivatives of these
    activations below 2, so a difference is off by e^2 / 6 * 2 per unit of weight cubed, plus rounding / e."""
    from neurotensor_b200 import api
    gen = generator(11)
    x, w, b = randn(gen, 4, 6), randn(gen, 6, 5, scale=0.4), randn(gen, 5)
    gy = randn(gen, 4, 5)
    _, pre = api.linear_act(x, w, b, act, want_pre=True)
    gx, gw, gb = api.linear_act_backward(x, w, pre, gy, act)
    e = 2.0 ** -6

    def loss(x, w, b):
        return float((api.linear_act(x, w, b, act).double() * gy.double()).sum())

    for t, g in ((x, gx), (w, gw), (b, gb)):
        for at in range(0, t.numel(), 3):
            up, down = t.clone(), t.clone()
            up.view(-1)[at] += e
            down.view(-1)[at] -= e
            args = [[v if v is not t else s for v in (x, w, b)] for s in (up, down)]
            d = (loss(*args[0]) - loss(*args[1])) / (2 * e)
            reach = float(gy.abs().sum()) * max(1.0, float(x.abs().max()), float(w.abs().max())) ** 3
            assert abs(d - float(g.reshape(-1)[at])) <= e * e / 3 * reach + 2.0 ** -20 / e * reach


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (3, 7, 5), (8, 512, 256), (33, 100, 130), (129, 272, 200), (300, 641, 513), (1, 4096, 4096), (16, 4096, 2048),
                                   (1100, 144, 1040), (2600, 80, 4104)])
def test_linear_int8(m, k, n, dtype, act):
    from neurotensor_b200 import api
    gen = generator(m + 7 * k + 31 * n)
    q = torch.randint(-127, 128, (m, k), generator=gen, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (k, n), generator=gen, device="cuda", dtype=torch.int8)
    s = torch.rand(m, generator=gen, device="cuda") * 0.02 + 0.001
    ws = (torch.rand(n, generator=gen, device="cuda") * 0.02 + 0.001) / math.sqrt(k)
    b = randn(gen, n, dtype=dtype) if m % 2 else None
    r = randn(gen, m, n, dtype=dtype) if n % 2 == 0 else None
    exact = (q.double() @ w.double()) * s.double()[:, None] * ws.double()
    z64 = exact + (b.double() if b is not None else 0)
    v64, _ = act64(z64, act)
    y64 = v64 + (r.double() if r is not None else 0)
    tol = half_step(dtype) * y64.abs() * (1 + 2.0 ** -9) + 1.13 * 2.0 ** -21 * (exact.abs() + (b.double().abs() if b is not None else 0)) + \
        2.0 ** -20 * (v64.abs() + z64.abs() * 2.0 ** -3) + 2.0 ** -23 * y64.abs() + smallest(dtype)
    for transpose in (False, True):
        wt = w.t().contiguous() if transpose else w
        y = api.linear_int8(q, s, wt, ws, b, act, residual=r, transpose_w=transpose, dtype=dtype)
        within(y, y64, tol, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_activations_far_out(act, dtype):
    """Values far from zero through a product with the identity: no overflow on the way, tails that keep their sign."""
    from neurotensor_b200 import api
    z = torch.tensor([[0.0, -0.0, 1e-6, -1e-6, 3.0, -3.0, 9.0, -9.0, 30.0, -30.0, 300.0, -300.0, 6e4, -6e4, 0.5, -0.5]], device="cuda").to(dtype)
    eye = torch.eye(16, device="cuda", dtype=dtype)
    y, pre = api.linear_act(z, eye, None, act, want_pre=True)
    assert torch.equal(pre, z)
    v64, slope = act64(z.double(), act)
    tail = 2.0 ** -17 if dtype == F32 else 2.0 ** -12          # e^-u for u up to 90: the argument's rounding, 90 2^-24, and its scale
    within(y, v64, (half_step(dtype) * (1 + 2.0 ** -9) + tail) * v64.abs() + 2 * smallest(dtype) + 2.0 ** -126, "value")
    gx, _, _ = api.linear_act_backward(z, eye, pre, torch.ones_like(z), act)
    within(gx, slope, (half_step(dtype) * (1 + 2.0 ** -9) + tail) * slope.abs() + 2.0 ** -19 + 2 * smallest(dtype), "slope")


@pytest.mark.gpu
def test_linear_layouts():
    """Leading dims, padded and misaligned rows, the residual's own place, a residual with padded rows, empty calls."""
    from neurotensor_b200 import _lib, api
    gen = generator(3)
    for dtype in (F16, F32):
        w, b = randn(gen, 96, 72, scale=0.1, dtype=dtype), randn(gen, 72, dtype=dtype)
        big, rbig = randn(gen, 5, 30, 120, dtype=dtype), randn(gen, 5, 30, 90, dtype=dtype)
        for x, r in ((big[..., :96], rbig[..., :72]), (big[..., 3:99], rbig[..., 1:73]), (big[:, 3, 8:104], rbig[:, 3, 8:80]),
                     (big[1, 2, :96], rbig[1, 2, :72]), (big.transpose(0, 1)[..., :96], rbig.transpose(0, 1)[..., :72])):
            y, pre = api.linear_act(x, w, b, "silu", residual=r, want_pre=True)
            ref = api.linear_act(x.contiguous(), w, b, "silu", residual=r.contiguous(), want_pre=True)
            assert torch.equal(y, ref[0]) and torch.equal(pre, ref[1]) and y.shape == x.shape[:-1] + (72,)
            got = api.linear_act_backward(x, w, pre, r, "silu")
            ref = api.linear_act_backward(x.contiguous(), w, pre, r.contiguous(), "silu")
            assert all(torch.equal(p, q) for p, q in zip(got, ref)) and got[0].shape == x.shape
        # y in the residual's place, padded rows: the padding stays as it was
        x = big[0, :, :96]
        place = rbig[0].clone()
        want = api.linear_act(x, w, b, "gelu", residual=place[:, :72])
        d, _, keep, _ = api._linear_desc("linear_act", x, w, b, "gelu", place[:, :72], False, dtype)
        d.y, d.y_row_stride = place.data_ptr(), 90
        need = _lib.lib().ntb200_linear_act_workspace_bytes(ctypes.byref(d))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        _lib.check(_lib.lib().ntb200_linear_act(ctypes.byref(d), ws.data_ptr(), need, api._stream()))
        assert torch.equal(place[:, :72], want) and torch.equal(place[:, 72:], rbig[0][:, 72:])
        # nothing to do, and nothing to sum: y = act(bias) + residual
        assert api.linear_act(big[:0, 0, :96], w, b, "gelu").shape == (0, 72)
        y = api.linear_act(torch.empty(3, 0, device="cuda", dtype=dtype), torch.empty(0, 72, device="cuda", dtype=dtype), b, "relu")
        assert torch.equal(y, torch.clamp(b, min=0).expand(3, 72))
        gx, gw, gb = api.linear_act_backward(big[:0, 0, :96], w, torch.empty(0, 72, device="cuda", dtype=dtype),
                                             torch.empty(0, 72, device="cuda", dtype=dtype), "gelu")
        assert gx.shape == (0, 96) and not bool(gw.any()) and not bool(gb.any())


@pytest.mark.gpu
@pytest.mark.parametrize("ex,ew", [(100, 20), (-70, -50), (120, -120), (-100, 90)])
@pytest.mark.parametrize("n", [1024, 1001])
def test_linear_float32_range(n, ex, ew):
    """Float32 operands far from 1: the product of their scales leaves the type's range, their products do not."""
    from neurotensor_b200 import api
    gen = generator(ex)
    x, w = randn(gen, 256, 512), randn(gen, 512, n)
    x[3], w[:, 5] = 0.0, 0.0
    x[4, :256], w[256:, 6] = 0.0, 0.0                       # a sum of nothing but zeros
    want = api.linear_act(x, w)
    got = api.linear_act(x * 2.0 ** ex, w * 2.0 ** ew)
    # Powers of two change no digit, and the results are the same: but a weight below 2^-126 is rounded to a multiple of
    # 2^-149 before the call.  Then the exact sums differ by |x| . lost, and each side's are off by 2^-21 |x| . |w| at most
    # (2^-22 from the parts of the operands, the rest fp32 sums of 512 terms that cancel at random).
    lost = ((w * 2.0 ** ew).double() * 2.0 ** -ew - w.double()).abs()
    slack = (x.double().abs() @ lost + 2.0 ** -20 * (x.double().abs() @ w.double().abs())) * float(lost.max() > 0)
    assert float(lost.max()) == 0 or ew == -120
    within(got.double() * 2.0 ** -(ex + ew), want.double(), slack, "scaled")
    big, small = torch.zeros(256, 512, device="cuda"), torch.zeros(512, n, device="cuda")
    big[:, 0], small[1] = 2.0 ** 120, 2.0 ** 120
    assert torch.equal(api.linear_act(big, small), torch.zeros(256, n, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_unusual_weights(dtype):
    """Weights that repeat one row, that skip elements, and that are windows of a larger matrix."""
    from neurotensor_b200 import api
    gen = generator(41)
    big, x = randn(gen, 200, 300, scale=0.1, dtype=dtype), randn(gen, 70, 64, dtype=dtype)
    for w in (big[0, :96].expand(64, 96), big[:64, 0:288:3], big[1:129:2, 3:99], big[:96, :64].t(), big[:192:3, 5]):
        w = w if w.dim() == 2 else w[:, None].expand(64, 96)
        want = api.linear_act(x, w.contiguous(), None, "relu", want_pre=True)
        got = api.linear_act(x, w, None, "relu", want_pre=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a, b = api.linear_act_backward(x, w, got[1], got[0], "relu"), api.linear_act_backward(x, w.contiguous(), got[1], got[0], "relu")
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_two_streams_at_once():
    """The same operators on two streams and from two host threads, each with its own inputs."""
    import threading
    from neurotensor_b200 import api
    args = [block_inputs(generator(s), BF16, rows=200) for s in (51, 52)]
    want = [block_step(api, *a, "silu") for a in args]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[k] = block_step(api, *args[k], "silu")
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # pragma: no cover
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for k in (0, 1):
        assert all(torch.equal(got[k][n], want[k][n]) for n in want[k])


@pytest.mark.gpu
def test_linear_needs_its_workspace():
    from neurotensor_b200 import _lib, api
    x, w = torch.zeros(64, 33, dtype=F16, device="cuda"), torch.zeros(33, 40, dtype=F16, device="cuda")
    d, _, keep, _ = api._linear_desc("linear_act", x, w, None, "none", None, False, F16)
    y = torch.empty(64, 40, dtype=F16, device="cuda")
    d.y, d.y_row_stride = y.data_ptr(), 40
    assert _lib.lib().ntb200_linear_act_workspace_bytes(ctypes.byref(d)) >= 64 * 40 * 2
    assert _lib.lib().ntb200_linear_act(ctypes.byref(d), None, 0, api._stream()) == _lib.ERR_ALLOC
    assert b"workspace" in _lib.lib().ntb200_last_error_string()


# ---- distillation ---------------------------------------------------------------------------------------------------

def distill64(s, t, i, T, rw):
    rows, vocab = s.shape
    lq = torch.log_softmax(s.double() / T, 1)
    there = (i >= 0) & (i < vocab) & (t > -math.inf)
    row = torch.zeros(rows, dtype=torch.float64, device="cuda")
    grad = torch.zeros_like(lq)
    size = torch.zeros_like(lq)
    for r in range(rows):
        if not bool(there[r].any()) or float(rw[r]) == 0:
            continue
        at = i[r][there[r]].long()
        p = torch.softmax(t[r][there[r]].double() / T, 0)
        full = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, at, p)
        row[r] = T * T * (torch.xlogy(p, p) - p * lq[r][at]).sum()
        c = float(rw[r]) * T
        grad[r] = c * (lq[r].exp() - full)
        size[r] = abs(c) * (lq[r].exp() + full)
    return (row * rw.double()).sum(), row, grad, size


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 5, 2), (9, 1000, 8), (5, 4099, 64), (4, 32000, 33), (2, 131072, 128), (3, 300001, 5), (2, 2048, 1024), (700, 257, 4),
                                            (1300, 1001, 40), (460, 40007, 7), (450, 131072, 64), (450, 98304, 128)])     # enough rows to stream
def test_distill(rows, vocab, top, dtype, T):
    from neurotensor_b200 import api
    gen = generator(rows + vocab + top)
    s = randn(gen, rows, vocab, scale=3.0, dtype=dtype)
    t = randn(gen, rows, top, scale=3.0, dtype=dtype)
    i = torch.randint(0, vocab, (rows, top), generator=gen, device="cuda", dtype=torch.int32)    # the same column twice among them
    if top > 2:
        i[:, 1] = i[:, 0]
        i[0, 2], t[-1, 2] = -1, -math.inf
    if rows > 2:
        i[1] = vocab + 7                                           # a row that has no entry
        s[2, vocab // 2:vocab // 2 + 1] = -math.inf                # a column that is masked out of the student
        i[2][i[2] == vocab // 2] = -1
    rw = torch.rand(rows, generator=gen, device="cuda") + 0.1
    if rows > 3:
        rw[3] = 0
        s[3, 0] = math.nan                                         # not read
    loss, row, grad = api.distill_topk(s, t, i, temperature=T, row_weight=rw)
    loss64, row64, grad64, size = distill64(s, t, i, T, rw)
    # the exponents reach 2^6, so their fp32 rounding is 2^-18 of each probability; sums of vocab terms add their own
    e = 2.0 ** -17 + 2.0 ** -24 * min(vocab, 4096)
    within(grad, grad64, half_step(dtype) * grad64.abs() * (1 + 2.0 ** -9) + e * size + smallest(dtype), "grad")
    scale = T * T * (1 + float(s[torch.isfinite(s)].abs().max()) * 2 / T + float(t[torch.isfinite(t)].abs().max()) * 2 / T + math.log(vocab + 1))
    within(row, row64, e * scale * torch.ones_like(row64), "row")
    within(loss, loss64, e * scale * float(rw.sum()) + rows * 2.0 ** -24 * float((row64.abs() * rw).sum()), "loss")
    again = api.distill_topk(s, t, i.long(), temperature=T, row_weight=rw)
    assert torch.equal(again[0], loss) and torch.equal(again[1], row) and torch.equal(again[2], grad)
    only = api.distill_topk(s, t, i, temperature=T, row_weight=rw, want_grad=False)
    assert only[2] is None and torch.equal(only[1], row)
    place = s.clone()
    loss2, _, g2 = api.distill_topk(place, t, i, temperature=T, row_weight=rw, out_grad=place)
    assert g2 is place and torch.equal(place, grad) and torch.equal(loss2, loss)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [64, 1001, 40000, 131072, 400001])
def test_distill_masked_by_the_lowest_value(vocab, dtype):
    """Columns masked out of the student by the type's lowest value: half of a row, all of it, and one the teacher names."""
    from neurotensor_b200 import api
    gen = generator(vocab)
    lowest = torch.finfo(dtype).min
    s = randn(gen, 6, vocab, scale=3.0, dtype=dtype)
    t, i = randn(gen, 6, 4, scale=2.0), torch.randint(0, vocab // 2, (6, 4), generator=gen, device="cuda")
    s[1:4, vocab // 2:] = lowest
    s[0] = lowest
    s[4, :vocab - 1] = lowest
    i[4] = vocab - 1
    i[2, 1] = vocab - 1
    i[5] = -1
    rw = torch.full((6,), 0.125, device="cuda")
    loss, row, grad = api.distill_topk(s, t, i, row_weight=rw)
    loss64, row64, grad64, size = distill64(s, t, i, 1.0, rw)
    e = 2.0 ** -17 + 2.0 ** -24 * min(vocab, 4096)
    within(grad, grad64, half_step(dtype) * grad64.abs() * (1 + 2.0 ** -9) + e * size + smallest(dtype), "grad")
    within(row, row64, e * (row64.abs() + 100), "row")     # the others' logits and logarithms stay below 50
    within(loss, loss64, e * (loss64.abs() + 100), "loss")


@pytest.mark.gpu
def test_distill_layouts_and_mean():
    from neurotensor_b200 import api
    gen = generator(8)
    big = randn(gen, 4, 6, 200, dtype=BF16)
    t, i = randn(gen, 4, 6, 5, dtype=F32), torch.randint(0, 128, (4, 6, 5), generator=gen, device="cuda")
    for s in (big[..., :128], big[..., 1:129], big[..., 8:136]):
        loss, row, grad = api.distill_topk(s, t, i)                 # the default weight is the mean over rows
        ref = api.distill_topk(s.contiguous(), t, i, row_weight=torch.full((4, 6), 1 / 24, device="cuda"))
        assert same_but_order(grad, ref[2]) and same_but_order(row, ref[1]) and same_but_order(loss, ref[0]) and grad.shape == s.shape
    loss, row, grad = api.distill_topk(big[:0, :, :128], t[:0], i[:0])
    assert float(loss) == 0 and row.shape == (0, 6) and grad.shape == (0, 6, 128)
    # the gradient is the difference quotient of the loss: step e, third derivatives of log-sum-exp below 1
    s = randn(gen, 2, 40)
    t, i = randn(gen, 2, 3), torch.randint(0, 40, (2, 3), generator=gen, device="cuda")
    _, _, g = api.distill_topk(s, t, i, temperature=1.5)
    e = 2.0 ** -5
    for at in range(0, 80, 7):
        up, down = s.clone(), s.clone()
        up.view(-1)[at] += e
        down.view(-1)[at] -= e
        d = (float(api.distill_topk(up, t, i, temperature=1.5)[0]) - float(api.distill_topk(down, t, i, temperature=1.5)[0])) / (2 * e)
        assert abs(d - float(g.view(-1)[at])) <= e * e / 6 * 1.5 + 2.0 ** -19 / e


# ---- together, as they are used -------------------------------------------------------------------------------------

def block_inputs(gen, dtype, rows=70, width=64, hidden=136, vocab=500, top=6):
    p = dict(n1=(1 + randn(gen, width, scale=0.2)).to(dtype), w1=randn(gen, width, hidden, scale=width ** -0.5, dtype=dtype),
             b1=randn(gen, hidden, scale=0.2, dtype=dtype), w2=randn(gen, hidden, width, scale=hidden ** -0.5, dtype=dtype),
             b2=randn(gen, width, scale=0.2, dtype=dtype), n2=(1 + randn(gen, width, scale=0.2)).to(dtype),
             head=randn(gen, width, vocab, scale=2 * width ** -0.5, dtype=dtype))
    x, stream = randn(gen, rows, width, dtype=dtype), randn(gen, rows, width, scale=2.0, dtype=dtype)
    t = randn(gen, rows, top, scale=2.0, dtype=dtype)
    i = torch.randint(0, vocab, (rows, top), generator=gen, device="cuda", dtype=torch.int32)
    rw = torch.full((rows,), 1.0 / rows, device="cuda")
    return p, x, stream, t, i, rw


def block_step(api, p, x, stream, t, i, rw, act):
    """Norm with residual, two linears around an activation, the second with the residual, norm, head, loss; and back."""
    y1, h1, s1 = api.rms_norm(x, p["n1"], residual=stream)
    a, pre = api.linear_act(y1, p["w1"], p["b1"], act, want_pre=True)
    h2 = api.linear_act(a, p["w2"], p["b2"], residual=h1)
    y2, _, s2 = api.rms_norm(h2, p["n2"])
    logits = api.linear_act(y2, p["head"])
    loss, _, g = api.distill_topk(logits, t, i, temperature=2.0, row_weight=rw)
    out = {"loss": loss, "logits": logits}
    gy2, out["head"], _ = api.linear_act_backward(y2, p["head"], None, g, want_bias=False)
    gh2, out["n2"] = api.rms_norm_backward(h2, p["n2"], s2, gy2)
    ga, out["w2"], out["b2"] = api.linear_act_backward(a, p["w2"], None, gh2)
    gy1, out["w1"], out["b1"] = api.linear_act_backward(y1, p["w1"], pre, ga, act)
    out["x"], out["n1"] = api.rms_norm_backward(h1, p["n1"], s1, gy1, grad_h=gh2)
    return out


def block64(p, x, stream, t, i, rw, act):
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    x = x.double().requires_grad_()
    h1 = x + stream.double()
    norm = lambda h, w: h * (h.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
    a = act64(norm(h1, q["n1"]) @ q["w1"] + q["b1"], act)[0]
    h2 = a @ q["w2"] + q["b2"] + h1
    logits = norm(h2, q["n2"]) @ q["head"]
    lq = torch.log_softmax(logits / 2.0, 1)
    pt = torch.softmax(t.double() / 2.0, 1)
    loss = (rw.double() * 4.0 * (torch.xlogy(pt, pt) - pt * lq.gather(1, i.long())).sum(1)).sum()
    names = sorted(q)
    grads = torch.autograd.grad(loss, [x] + [q[k] for k in names])
    return dict(zip(["x"] + names, grads), loss=loss.detach(), logits=logits.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_block_forward_and_backward(dtype, act):
    """A training step through every operator.  Its tensors pass at most 10 roundings to the dtype on the way (y1, pre or
    a, h2, y2, logits, and five gradients back), each half a step at worst; by the norm of a tensor they add up to at most
    twice that through norms and activations of slope near 1."""
    from neurotensor_b200 import api
    args = block_inputs(generator(21), dtype)
    got, want = block_step(api, *args, act), block64(*args, act)
    bound = 20 * half_step(dtype) if dtype != F32 else 2.0 ** -16
    if dtype == F16:   # the loss is a mean over 70 rows and 500 columns: its smallest gradients are subnormal
        bound += 500 * smallest(F16) / float(want["logits"].std())
    for k, v in want.items():
        d = float((got[k].double() - v).norm() / v.norm())
        assert d <= bound, (k, d, bound)


@pytest.mark.gpu
def test_block_served_in_int8():
    """The same block in 8 bits against 64 bits on the quantised values themselves, so that only roundings remain."""
    from neurotensor_b200 import api
    p, x, stream, _, _, _ = block_inputs(generator(22), BF16)
    w1, s1 = api.quantize_rows(p["w1"].t().contiguous())
    w2, s2 = api.quantize_rows(p["w2"].t().contiguous())
    q, sc, h1 = api.rms_norm_int8(x, p["n1"], residual=stream)
    a = api.linear_int8(q, sc, w1, s1, p["b1"], "gelu", transpose_w=True)
    qa, sa = api.quantize_rows(a)
    h2 = api.linear_int8(qa, sa, w2, s2, p["b2"], residual=h1, transpose_w=True)
    u = half_step(BF16) * (1 + 2.0 ** -8)
    a64 = act64((q.double() * sc.double()[:, None]) @ (w1.double() * s1.double()[:, None]).t() + p["b1"].double(), "gelu")[0]
    within(a, a64, u * a64.abs() + 2.0 ** -17, "hidden")
    h64 = (qa.double() * sa.double()[:, None]) @ (w2.double() * s2.double()[:, None]).t() + p["b2"].double() + h1.double()
    within(h2, h64, u * h64.abs() + 2.0 ** -17, "stream")
    full = act64(block_norm(x, stream, p["n1"]) @ p["w1"].double() + p["b1"].double(), "gelu")[0] @ p["w2"].double() + p["b2"].double() + x.double() + stream.double()
    assert float((h2.double() - full).norm() / full.norm()) < 4 / 127     # four quantisations of half a step of 1 / 127 of a row's maximum


def block_norm(x, stream, w):
    h = x.double() + stream.double()
    return h * (h.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()


@pytest.mark.gpu
def test_block_captured_and_on_another_stream():
    """The step captured into two graphs of one stream, replayed on two others at once, beside eager calls: workspaces
    belong to the calls, so nothing is shared."""
    from neurotensor_b200 import api
    args = [block_inputs(generator(s), BF16, rows=150) for s in (31, 32)]
    want = [block_step(api, *a, "gelu") for a in args]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for a in args:
            block_step(api, *a, "gelu")
        side.synchronize()
        for a in args:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = block_step(api, *a, "gelu")
            graphs.append((g, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = block_step(api, *args[0], "gelu")
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert all(torch.equal(out[k], w[k]) for k in w)
    assert all(torch.equal(eager[k], want[0][k]) for k in eager)
