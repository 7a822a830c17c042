"""GPU: RMS norm with the residual's addition, 8-bit block-scaled products and rotary positions against their definitions in 64 bits.

Tolerances.  A result that is rounded to a type is off by half a step of it, eps/2 of the value (bf16 2^-8, fp32 2^-24, e4m3 2^-4 or
2^-10 of the scale below its normal range).  Before that rounding the kernels compute in fp32; the allowances below count the
roundings of each formula (U = 2^-24).
"""
import math

import pytest
import torch

from get_model_amd import functional as Fn
from get_model_amd import kernels as K

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F32: U}


def rnd(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def within(got, ref, tol, what=""):
    """|got - ref| <= tol element by element; NaN and infinities in the same places."""
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(got)), what
    d = ((got - ref).abs() - tol)[fin]
    assert d.numel() == 0 or d.max().item() <= 0, f"{what}: {d.max().item():.3g} over the tolerance"


def norm_ref(x, w, res, eps):
    h = x.double() if res is None else x.double() + res.double()
    rstd = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return h, rstd, h * rstd * w.double()


# relative error of y before its rounding: h (1 U), the squares' sum (each lane adds at most 16 + 6 + 16 terms of one sign: 40 U,
# halved by the root), division and root (3 U), two products (2 U)
Y_REL = 32 * U

WIDTHS = [1, 3, 64, 127, 128, 283, 768, 1000, 1028, 2304, 5000, 8192, 16384]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("M,xt,rt,yt", [(1, BF16, F32, BF16), (5, F32, None, F32), (600, BF16, BF16, F32), (67, F32, F32, BF16), (515, BF16, None, BF16)])
def test_rms_norm_forward(D, M, xt, rt, yt):
    x, w = rnd(M, D, seed=1, dtype=xt), 1 + 0.3 * rnd(D, seed=2)
    res = None if rt is None else rnd(M, D, seed=3, dtype=rt, scale=2.0)
    y, h, rstd = K.rms_norm_fwd(x, w, res, 1e-5, yt, want_rstd=True)
    rh, rrstd, ry = norm_ref(x, w, res, 1e-5)
    # where x and the residual cancel, the sum's one rounding is relative to itself: fp32 sums of bf16 / fp32 values
    within(y, ry, ry.abs() * (HALF[yt] + Y_REL) + 1e-30, "y")
    within(rstd, rrstd[:, 0], rrstd[:, 0] * Y_REL, "rstd")
    assert y.dtype == yt and rstd.dtype == F32
    if rt is None:
        assert h is None
    else:
        within(h, rh, rh.abs() * (HALF[rt] + (U if rt is not F32 else 0)), "h")


@pytest.mark.parametrize("D", [1, 127, 283, 768, 1500, 2048, 2052, 8192])
@pytest.mark.parametrize("M,xt,rt,yt", [(1, BF16, F32, BF16), (5, F32, None, F32), (3000, BF16, BF16, BF16), (1300, F32, F32, BF16), (515, BF16, None, F32)])
def test_rms_norm_backward_formula(D, M, xt, rt, yt):
    x, w = rnd(M, D, seed=1, dtype=xt).requires_grad_(), (1 + 0.3 * rnd(D, seed=2)).requires_grad_()
    res = None if rt is None else rnd(M, D, seed=3, dtype=rt).requires_grad_()
    dy = rnd(M, D, seed=4, dtype=yt)
    out = Fn.rms_norm(x, w, res, 1e-5, yt)
    if rt is None:
        dx, dw = torch.autograd.grad(out, (x, w), dy)
        dh, stored, dr = None, x.detach().double(), None
    else:
        dh = rnd(M, D, seed=5, dtype=rt)
        dx, dw, dr = torch.autograd.grad(out, (x, w, res), (dy, dh))
        stored = out[1].detach().double()        # the backward works on h as it is stored
    _, rstd, _ = norm_ref(x.detach(), w.detach(), None if res is None else res.detach(), 1e-5)
    hh, g = stored * rstd, dy.double() * w.detach().double()
    c = (g * hh).mean(1, keepdim=True)
    d = rstd * (g - hh * c) + (0 if dh is None else dh.double())
    # each term carries Y_REL; the mean's error is Y_REL of the mean of absolute values
    mean_abs = (g * hh).abs().mean(1, keepdim=True)
    slack = 2 * Y_REL * (rstd * (g.abs() + hh.abs() * (c.abs() + mean_abs)) + (0 if dh is None else dh.double().abs()))
    within(dx, d, d.abs() * HALF[xt] + slack, "dx")
    if dr is not None:
        within(dr, d, d.abs() * HALF[rt] + slack, "dresidual")
    # a column's sum: at most M/512 + 16 terms in a chain, then fixed trees of 64
    p = (dy.double() * hh).abs().sum(0)
    within(dw, (dy.double() * hh).sum(0), p * (M / 512 + 96) * U, "dw")


def test_rms_norm_gradient_against_differences():
    M, D = 7, 300
    x, w, res = rnd(M, D, seed=1), 1 + 0.3 * rnd(D, seed=2), rnd(M, D, seed=3)
    dy, dh = rnd(M, D, seed=4).double(), rnd(M, D, seed=5).double()
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    grads = torch.autograd.grad(Fn.rms_norm(leaves[0], leaves[1], leaves[2], out_dtype=F32), leaves, (dy.float(), dh.float()))

    def value(x, w, res):
        y, h = Fn.rms_norm(x, w, res, out_dtype=F32)
        return (y.double() * dy).sum() + (h.double() * dh).sum()
    e = 2.0 ** -7
    for i, g in enumerate(grads):
        v = rnd(*g.shape, seed=6 + i)
        up, down = [list((x, w, res)) for _ in range(2)]
        up[i], down[i] = up[i] + e * v, down[i] - e * v
        slope = (value(*up) - value(*down)) / (2 * e)
        want = (g.double() * v.double()).sum()
        # the difference's own error: e^2/6 times the third derivative along v (y's is below 15 times its size per unit of v / rms)
        # and the values' fp32 error over 2e
        size = (g.double().abs() * v.double().abs()).sum()
        assert abs(slope - want) <= 15 * e * e / 6 * size + 64 * U / (2 * e) * (M * D) ** 0.5 * 8, i


def test_rms_norm_strides_shapes_and_one_output_only():
    wide = rnd(40, 1000, seed=1)
    x, w = wide[:, 3:771], 1 + 0.3 * rnd(768, seed=2)                 # rows apart, off 16 bytes
    y, _, _ = K.rms_norm_fwd(x, w)
    assert torch.equal(y, K.rms_norm_fwd(x.contiguous(), w)[0])
    # [B, T, D] with a transposed batch, and an expanded row
    t = rnd(6, 5, 768, seed=3).transpose(0, 1)
    assert torch.equal(Fn.rms_norm(t, w), Fn.rms_norm(t.contiguous(), w))
    one = rnd(1, 768, seed=4)
    assert torch.equal(Fn.rms_norm(one.expand(9, 768), w), Fn.rms_norm(one, w).expand(9, 768))
    row = one.clone().requires_grad_()
    Fn.rms_norm(row.expand(9, 768), w, out_dtype=F32).backward(torch.ones(9, 768, device="cuda"))
    alone = one.clone().requires_grad_()
    Fn.rms_norm(alone, w, out_dtype=F32).backward(torch.ones(1, 768, device="cuda"))
    within(row.grad, 9 * alone.grad.double(), 9 * 16 * U * alone.grad.abs().double() + 1e-9)      # nine equal terms, added in fp32
    # a gradient for one of the outputs alone
    x, res = rnd(4, 96, seed=5, dtype=BF16).requires_grad_(), rnd(4, 96, seed=6).requires_grad_()
    w = torch.ones(96, device="cuda", requires_grad=True)
    y, h = Fn.rms_norm(x, w, res)
    g = rnd(4, 96, seed=7)
    gx, gw, gr = torch.autograd.grad(h, (x, w, res), g, retain_graph=True)
    assert torch.equal(gr, g) and torch.equal(gx, g.to(BF16)) and not gw.any()
    ones = torch.ones_like(y)
    only_y = torch.autograd.grad(y, (x, w, res), ones, retain_graph=True)
    both = torch.autograd.grad((y, h), (x, w, res), (ones, torch.zeros_like(h)))
    assert all(torch.equal(a, b) for a, b in zip(only_y, both))
    # no rows
    e = Fn.rms_norm(torch.zeros(0, 96, device="cuda", requires_grad=True), w, out_dtype=F32)
    assert e.shape == (0, 96)
    e.sum().backward()
    assert not w.grad.any()


def test_rms_norm_rows_that_are_not_finite_stay_alone():
    x, w = rnd(9, 768, seed=1), torch.ones(768, device="cuda")
    want = K.rms_norm_fwd(x, w, out_dtype=F32)[0]
    bad = x.clone()
    bad[2, 5], bad[4, 700], bad[6] = float("nan"), float("inf"), 0.0
    y = K.rms_norm_fwd(bad, w, out_dtype=F32)[0]
    keep = torch.tensor([0, 1, 3, 5, 7, 8], device="cuda")
    assert torch.equal(y[keep], want[keep]) and y[2].isnan().all() and y[4, 700].isnan() and not y[6].any()
    q, s, _ = K.rms_norm_fp8(bad, w)
    v = q.float()
    assert torch.isfinite(v[keep]).all() and v[2].isnan().all()
    assert v[4, 640:768].isnan().all() and not v[4, :640].any()       # the infinite value's block; finite / inf = 0 elsewhere
    assert not v[6].any() and bool((s.view(torch.uint8)[6] == 127).all())


# ---------------------------------------------------------------------------------------------------------------- 8 bits
def scale_of(amax):
    """The smallest power of two with amax <= 448 * scale, in 64 bits; 1 for zero, at least 2^-126."""
    m, e = torch.frexp(amax.double())
    e = (e - 9 + (m > 0.875).int()).clamp(min=-126)
    return torch.where(amax == 0, torch.ones_like(amax, dtype=F64), torch.exp2(e.double()))


def blocks(v, rows=1):
    R, C = v.shape
    p = torch.nn.functional.pad(v, (0, -C % 128, 0, -R % rows))
    return p.view(p.shape[0] // rows, rows, p.shape[1] // 128, 128)


def values(q, s, rows=1):
    f = s.view(torch.uint8).double() - 127
    return q.double() * torch.exp2(f).repeat_interleave(128, 1).repeat_interleave(rows, 0)[:q.shape[0]]


@pytest.mark.parametrize("M,D", [(1, 1), (3, 127), (5, 128), (600, 283), (1, 768), (515, 768), (66, 1000), (2, 5000), (3, 16384)])
@pytest.mark.parametrize("xt", [BF16, F32])
def test_quant_rows_is_exact(M, D, xt):
    x = rnd(M, D, seed=1, dtype=xt) * torch.exp(3 * rnd(M, 1, seed=2)).to(xt)
    x[0] = 0
    if M > 2:
        x[1], x[2] = 448.0, 449.0
    q, s = K.quant_rows_fp8(x)
    b = blocks(x.double())
    want = scale_of(b.abs().amax((1, 3)))
    assert torch.equal(torch.exp2(s.view(torch.uint8).double() - 127), want)
    exact = (b / want[:, None, :, None]).view(M, -1)
    assert torch.equal(q.view(torch.uint8), exact.float().to(torch.float8_e4m3fn).view(torch.uint8))      # scaled exactly, rounded once


@pytest.mark.parametrize("N,D", [(1, 1), (128, 128), (129, 130), (768, 768), (2304, 768), (1000, 283)])
@pytest.mark.parametrize("wt", [BF16, F32])
def test_quant_blocks_is_exact(N, D, wt):
    w = rnd(N, D, seed=1, dtype=wt, scale=0.05)
    q, s = K.quant_blocks_fp8(w)
    b = blocks(w.double(), 128)
    want = scale_of(b.abs().amax((1, 3)))
    assert torch.equal(torch.exp2(s.view(torch.uint8).double() - 127), want)
    exact = (b / want[:, None, :, None]).view(-1, b.shape[2] * 128)[:N]
    assert torch.equal(q.view(torch.uint8), exact.float().to(torch.float8_e4m3fn).view(torch.uint8))


def test_quantisation_of_extremes():
    x = torch.zeros(6, 256, device="cuda")
    x[0, 3], x[1, 200], x[2, 0], x[3, 1], x[4, 2], x[5, 7] = float("inf"), float("nan"), 3e38, 1e-38, 2.0 ** -149, -3e38
    x[:, 130] = 1.0
    q, s = K.quant_rows_fp8(x)
    v = values(q, s)
    assert v[0, :128].isnan().all() and v[1, 128:].isnan().all() and bool((v[0, 130:131] == 1).all())
    assert abs(v[2, 0].item() / 3e38 - 1) <= 2 ** -4 and abs(v[5, 7].item() / -3e38 - 1) <= 2 ** -4
    # below 2^-126 * 448 the scale stays at 2^-126: the value is off by half a step of the subnormal range, 2^-10 * 2^-126
    assert abs(v[3, 1].item() - 1e-38) <= 1e-38 * 2 ** -4 and abs(v[4, 2].item() - 2.0 ** -149) <= 2.0 ** -136
    strided = rnd(20, 300, seed=1)[:, 1:270]
    a, b = K.quant_rows_fp8(strided), K.quant_rows_fp8(strided.contiguous())
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1].view(torch.uint8), b[1].view(torch.uint8))
    assert K.quant_rows_fp8(x[:0])[0].shape == (0, 256)


@pytest.mark.parametrize("M,D", [(1, 768), (600, 768), (5, 283), (1030, 128), (3, 8192), (1, 16384), (700, 1024)])
@pytest.mark.parametrize("xt,rt", [(BF16, F32), (F32, None), (BF16, BF16), (BF16, None), (F32, F32)])
def test_rms_norm_fp8(M, D, xt, rt):
    x, w = rnd(M, D, seed=1, dtype=xt), 1 + 0.3 * rnd(D, seed=2)
    res = None if rt is None else rnd(M, D, seed=3, dtype=rt)
    q, s, h = K.rms_norm_fp8(x, w, res, 1e-6)
    rh, _, ry = norm_ref(x, w, res, 1e-6)
    b = blocks(ry)
    amax = b.abs().amax((1, 3))
    scale = torch.exp2(s.view(torch.uint8).double() - 127)
    lo, hi = scale_of(amax * (1 - 2 * Y_REL)), scale_of(amax * (1 + 2 * Y_REL))      # next to a border either power is right
    assert bool(((scale == lo) | (scale == hi)).all())
    full = b.view(M, -1)
    v = values(q, s)
    # half a step of e4m3 (2^-4, or 2^-10 of the scale below its normal range) and y's own error
    tol = torch.maximum(full.abs() * 2.0 ** -4, scale.repeat_interleave(128, 1) * 2.0 ** -10) + full.abs() * 2 * Y_REL
    within(v, full, tol, "values")
    assert not q.view(torch.uint8)[:, D:].any()          # padding
    if rt is None:
        assert h is None
    else:
        within(h, rh, rh.abs() * (HALF[rt] + (U if rt is not F32 else 0)), "h")


def operands(M, N, Kd, seed=1):
    qa = K.quant_rows_fp8(rnd(M, Kd, seed=seed) * torch.exp(rnd(M, 1, seed=seed + 1)))
    return qa, K.quant_blocks_fp8(rnd(N, Kd, seed=seed + 2, scale=0.1))


def product_ref(qa, qb, bias):
    a, b = values(*qa), values(*qb, rows=128)
    out = torch.mm(a, b.t().contiguous())
    size = torch.mm(a.abs(), b.abs().t().contiguous())
    return (out if bias is None else out + bias.double()), size


# the matrix unit aligns a block's 128 products to the largest before it adds them and keeps at least 16 bits: 2^-15 of the
# absolute sum; the sum over blocks is fp32
PRODUCT_REL = 2.0 ** -15

SHAPES = [(1, 1, 1), (1, 17, 128), (1, 768, 768), (1, 2304, 300), (2, 130, 1000), (15, 64, 256), (16, 768, 4096), (17, 129, 640),
          (33, 2304, 768), (64, 1024, 512), (65, 100, 384), (127, 255, 129), (201, 768, 768), (255, 768, 2304), (256, 256, 256),
          (257, 257, 257), (300, 1000, 5000), (1000, 2304, 768), (2049, 513, 128), (4020, 768, 768), (1, 5000, 8192), (7, 8192, 1024),
          (700, 4096, 1024), (8000, 8, 256), (3, 3, 16384),
          # large tiles: few and many of them per CU, two to twenty blocks deep, ragged rows and columns, rows off 16 bytes
          (4096, 1024, 256), (2100, 2056, 384), (5000, 2304, 768), (20000, 1024, 256), (20001, 1000, 500), (16500, 2304, 512),
          (3000, 1501, 640), (9001, 1283, 256), (4100, 1025, 2600), (1111, 5003, 300), (20000, 370, 730),
          (13000, 1026, 300), (26000, 513, 384),
          # the depth split in two and in four, and the shapes next to those; two row groups of either operand
          (64, 300, 8192), (100, 767, 8200), (40, 8192, 6144), (33, 5001, 6272), (64, 2048, 6016), (12, 8200, 1024), (9, 8193, 300),
          (32, 4096, 700), (20, 33, 9000), (31, 8192, 256),
          # just over a round of large tiles: the last rows go to small ones
          (33000, 512, 1024), (32900, 511, 1100), (57600, 300, 1000)]


@pytest.mark.parametrize("M,N,Kd", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_gemm_fp8(M, N, Kd, bias):
    qa, qb = operands(M, N, Kd)
    b = rnd(N, seed=9) if bias else None
    got = K.gemm_fp8(*qa, *qb, bias=b)
    ref, size = product_ref(qa, qb, b)
    assert got.dtype == BF16
    within(got, ref, ref.abs() * HALF[BF16] + size * PRODUCT_REL + (0 if b is None else b.abs().double() * U), "product")


@pytest.mark.parametrize("M,N,Kd", [(1, 48, 256), (20, 33, 128), (130, 260, 384), (513, 768, 1024), (1025, 300, 640), (4097, 2305, 256), (12345, 1536, 1280)])
def test_gemm_fp8_of_small_integers(M, N, Kd):
    """Small whole numbers: every product and sum is exact, so a row, column or block out of place shows at once."""
    g = torch.Generator(device="cuda").manual_seed(5)
    a = torch.randint(-4, 5, (M, Kd), generator=g, device="cuda").float()
    b = torch.randint(-4, 5, (N, Kd), generator=g, device="cuda").float()
    ea = torch.randint(-2, 3, (M, Kd // 128), generator=g, device="cuda")
    eb = torch.randint(-2, 3, (-(-N // 128), Kd // 128), generator=g, device="cuda")

    def scales(e):
        t = torch.zeros(e.shape[0], (e.shape[1] + 3) // 4 * 4, dtype=torch.uint8, device="cuda")
        t[:, :e.shape[1]] = (e + 127).to(torch.uint8)
        return t.view(K.SCALE)[:, :e.shape[1]]
    qa, qb = (a.to(K.FP8), scales(ea)), (b.to(K.FP8), scales(eb))
    ref, _ = product_ref(qa, qb, None)
    assert torch.equal(K.gemm_fp8(*qa, *qb), ref.to(BF16))


def test_gemm_fp8_strided_rows_nan_rows_and_no_rows():
    M, N, Kd = 70, 200, 256
    qa, qb = operands(M, N, Kd)
    want = K.gemm_fp8(*qa, *qb)
    wide = torch.zeros(M, 400, dtype=torch.uint8, device="cuda").view(K.FP8)
    wide[:, 16:272].copy_(qa[0])
    pitch = torch.zeros(M, 12, dtype=torch.uint8, device="cuda").view(K.SCALE)
    pitch[:, 4:6].copy_(qa[1])
    assert torch.equal(K.gemm_fp8(wide[:, 16:272], pitch[:, 4:6], *qb), want)
    bad = qa[0].clone()
    bad.view(torch.uint8)[3, 100] = 0x7f
    got = K.gemm_fp8(bad, qa[1], *qb)
    keep = torch.arange(M, device="cuda") != 3
    assert got[3].isnan().all() and torch.equal(got[keep], want[keep])
    assert K.gemm_fp8(qa[0][:0], qa[1][:0], *qb).shape == (0, N)
    assert K.gemm_fp8(*qa, qb[0][:0], qb[1][:0]).shape == (M, 0)


@pytest.mark.parametrize("M,N,Kd", [(1, 1, 1), (1, 768, 768), (3, 130, 283), (16, 2304, 768), (9, 8200, 1000), (16, 64, 16384), (2, 33, 129), (5, 40, 8191)])
@pytest.mark.parametrize("xt", [BF16, F32])
def test_linear_of_few_rows_is_quantisation_and_product(M, N, Kd, xt):
    wide = rnd(M, Kd + 5, seed=1, dtype=xt) * torch.exp(2 * rnd(M, 1, seed=2)).to(xt)
    wide[0, :min(Kd, 128)] = 0
    qb, bias = K.quant_blocks_fp8(rnd(N, Kd, seed=3, scale=0.1)), rnd(N, seed=4)
    for x in (wide[:, :Kd], wide[:, 3:3 + Kd], wide[:, :Kd].contiguous(), wide[:1, :Kd].expand(M, Kd)):
        want = K.gemm_fp8(*K.quant_rows_fp8(x), *qb, bias)
        assert torch.equal(K.linear_rows_fp8(x, *qb, bias), want)
    if M > 1:
        bad = wide[:, :Kd].clone()
        bad[1, Kd - 1] = float("inf")
        got = K.linear_rows_fp8(bad, *qb)
        keep = torch.arange(M, device="cuda") != 1
        assert got[1].isnan().all() and torch.equal(got[keep], K.linear_rows_fp8(wide[:, :Kd], *qb)[keep])
    assert K.linear_rows_fp8(wide[:0, :Kd], *qb).shape == (0, N)


@pytest.mark.parametrize("M,N,Kd", [(1, 1, 1), (17, 768, 768), (64, 64, 128), (65, 130, 283), (201, 2304, 768), (100, 33, 1001), (31, 700, 5000), (4020, 256, 768), (70, 70, 9),
                                    (128, 65, 127), (129, 64, 1028)])
@pytest.mark.parametrize("xt", [BF16, F32])
def test_linear_in_tiles_is_quantisation_and_product(M, N, Kd, xt):
    wide = rnd(M, Kd + 5, seed=1, dtype=xt) * torch.exp(2 * rnd(M, 1, seed=2)).to(xt)
    wide[0, :min(Kd, 128)] = 0
    qb, bias = K.quant_blocks_fp8(rnd(N, Kd, seed=3, scale=0.1)), rnd(N, seed=4)
    for x in (wide[:, :Kd], wide[:, 3:3 + Kd], wide[:, :Kd].contiguous(), wide[:1, :Kd].expand(M, Kd)):
        assert torch.equal(K.linear_tiles_fp8(x, *qb, bias), K.gemm_fp8(*K.quant_rows_fp8(x), *qb, bias))
    if M > 1:
        bad = wide[:, :Kd].clone()
        bad[1, Kd - 1] = float("inf")
        got = K.linear_tiles_fp8(bad, *qb)
        keep = torch.arange(M, device="cuda") != 1
        assert got[1].isnan().all() and torch.equal(got[keep], K.linear_tiles_fp8(wide[:, :Kd], *qb)[keep])
    assert K.linear_tiles_fp8(wide[:0, :Kd], *qb).shape == (0, N)


def test_linear_fp8_takes_the_same_values_whatever_kernel_takes_it():
    w = torch.nn.Parameter(rnd(768, 768, seed=2, scale=0.1))
    x = rnd(9000, 768, seed=1, dtype=BF16)
    with torch.no_grad():
        whole = Fn.linear_fp8(x, w)
        for n in (1, 16, 17, 64, 1000, 4032, 4033, 8999):
            assert torch.equal(Fn.linear_fp8(x[:n], w), whole[:n]), n


def test_linear_fp8_and_its_weight_copy():
    x, w = rnd(2, 5, 300, seed=1, dtype=BF16), torch.nn.Parameter(rnd(140, 300, seed=2, scale=0.1))
    b = rnd(140, seed=3)
    with torch.no_grad():
        y = Fn.linear_fp8(x, w, b)
        qx, qw = K.quant_rows_fp8(x.view(10, 300)), K.quant_blocks_fp8(w)
        assert y.shape == (2, 5, 140) and torch.equal(y.view(10, 140), K.gemm_fp8(*qx, *qw, b))
        assert torch.equal(Fn.linear_fp8(qx, w, b), y.view(10, 140)) and torch.equal(Fn.linear_fp8(qx, qw, b), y.view(10, 140))
        assert torch.equal(Fn.linear_fp8(x[1, 2], w, b), y[1, 2])
        kept = Fn.w_fp8(w)[0]
        assert Fn.w_fp8(w)[0] is kept
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            z = Fn.linear_fp8(x, w, b)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(z, y)
        w.mul_(-1)       # the parameter changes: so does its copy
        assert torch.equal(Fn.linear_fp8(x, w), -Fn.linear_fp8(x, -w))
        assert Fn.w_fp8(w)[0] is not kept


# ---------------------------------------------------------------------------------------------------------------- rotary
def rotary_ref(x, inv, pos, layout, mag=1.0, sign=1.0):
    B, T, H, D = x.shape
    R = 2 * inv.numel()
    a = (pos.double().expand(B, T)[..., None] * inv)[:, :, None]
    c, s = mag * a.cos(), sign * mag * a.sin()
    t = x.double()
    if layout == "half":
        u, v = t[..., :R // 2], t[..., R // 2:R]
        out = torch.cat((u * c - v * s, v * c + u * s), -1)
        size = torch.cat((u.abs() + v.abs(),) * 2, -1)
    else:
        u, v = t[..., 0:R:2], t[..., 1:R:2]
        out = torch.stack((u * c - v * s, v * c + u * s), -1).flatten(-2)
        size = (u.abs() + v.abs()).repeat_interleave(2, -1)
    return torch.cat((out, t[..., R:]), -1), torch.cat((size * mag, torch.zeros_like(t[..., R:])), -1)


# cosine and sine: argument rounding below 1 U, polynomial and its roundings 3 U, magnitude 1 U; two products and a sum 2 U: 8 U of
# |u| + |v|, and 2^-52 of the angle (the reference's own rounding of the product)
def rotary_tol(ref, size, dtype, angle):
    return ref.abs() * HALF[dtype] + size * (8 * U + angle * 2.0 ** -51)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,D,R", [(1, 1, 1, 1, 2, 2), (64, 1, 12, 12, 64, 64), (2, 201, 12, 12, 64, 64), (3, 7, 5, 1, 96, 32), (2, 33, 4, 2, 80, 20),
                                           (1, 1000, 16, 2, 128, 64), (5, 3, 3, 3, 7, 6), (1, 2, 40, 40, 256, 256), (1, 3, 2, 1, 600, 520),
                                           (300, 17, 2, 2, 32, 16), (1, 1, 64, 8, 128, 128)])
def test_rotary(layout, dtype, B, T, Hq, Hk, D, R):
    packed = rnd(B, T, Hq + 2 * Hk, D, seed=1, dtype=dtype)
    q, k = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hk]
    inv = Fn.rotary_frequencies(R, device="cuda")[0]
    g = torch.Generator(device="cuda").manual_seed(3)
    pos = torch.randint(0, 100_000, (B, T), generator=g, device="cuda")
    qo, ko = Fn.rotary(q, k, inv, pos, layout=layout, magnitude=1.25)
    for got, x in ((qo, q), (ko, k)):
        ref, size = rotary_ref(x, inv, pos, layout, 1.25)
        within(got, ref, rotary_tol(ref, size, dtype, 1e5), "rotated")
        assert got.is_contiguous() and torch.equal(got[..., R:], x[..., R:])
    # int32 positions, one row of positions for all samples, an offset instead, q alone, in place
    assert torch.equal(Fn.rotary(q, k, inv, pos.int(), layout=layout, magnitude=1.25)[1], ko)
    line = torch.arange(5, 5 + T, device="cuda")
    by_line = Fn.rotary(q, None, inv, line, layout=layout)
    assert torch.equal(by_line, Fn.rotary(q, None, inv, offset=5, layout=layout))
    assert torch.equal(by_line, Fn.rotary(q, k, inv, line.expand(B, T), layout=layout)[0])
    inplace = packed.clone()
    Fn.rotary_(inplace[:, :, :Hq], inplace[:, :, Hq:Hq + Hk], inv, pos, layout=layout, magnitude=1.25)
    assert torch.equal(inplace[:, :, :Hq], qo) and torch.equal(inplace[:, :, Hq:Hq + Hk], ko)
    assert torch.equal(inplace[:, :, Hq + Hk:], packed[:, :, Hq + Hk:])          # the values are left as they were
    both = packed.clone()
    Fn.rotary_(both[:, :, :Hq + Hk], None, inv, pos, layout=layout, magnitude=1.25)
    assert torch.equal(both, inplace)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_far_positions(layout):
    """Base pairs, positions past 32 bits and before zero: the angle keeps its last bits."""
    pos = torch.tensor([0, 1, -1, 248_956_421, -7_000_001, 2 ** 31 + 5, 2 ** 33 + 1, 2 ** 40 - 3], device="cuda")
    x = rnd(1, 8, 2, 64, seed=1)
    inv = Fn.rotary_frequencies(64, device="cuda")[0]
    got = Fn.rotary(x, None, inv, pos, layout=layout)
    # the reference angle through integers: position * inv as an exact rational, reduced by pi to 200 bits
    from fractions import Fraction
    pi = Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)
    c, s = torch.zeros(8, 32, dtype=F64), torch.zeros(8, 32, dtype=F64)
    for i, p in enumerate(pos.tolist()):
        for j, f in enumerate(inv.tolist()):
            a = Fraction(f) * p
            a = float(a - 2 * pi * round(a / (2 * pi)))
            c[i, j], s[i, j] = math.cos(a), math.sin(a)
    c, s, t = c.cuda()[None, :, None], s.cuda()[None, :, None], x.double()
    u, v = (t[..., :32], t[..., 32:]) if layout == "half" else (t[..., 0::2], t[..., 1::2])
    pair = (u * c - v * s, v * c + u * s)
    ref = torch.cat(pair, -1) if layout == "half" else torch.stack(pair, -1).flatten(-2)
    size = torch.cat((u.abs() + v.abs(),) * 2, -1) if layout == "half" else (u.abs() + v.abs()).repeat_interleave(2, -1)
    within(got, ref, rotary_tol(ref, size, F32, 0.0), "far")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(layout):
    B, T, H, D = 2, 19, 3, 48
    inv, mag = Fn.rotary_frequencies(32, scaling="yarn", factor=4.0, original_length=512, device="cuda")
    pos = torch.arange(T, device="cuda") * 37
    q, k = rnd(B, T, H, D, seed=1).requires_grad_(), rnd(B, T, 1, D, seed=2).requires_grad_()
    gq, gk = rnd(B, T, H, D, seed=3), rnd(1, 1, 1, D, seed=4).expand(B, T, 1, D)      # a broadcast gradient
    qo, ko = Fn.rotary(q, k, inv, pos, layout=layout, magnitude=mag)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk), retain_graph=True)
    for got, g in ((dq, gq), (dk, gk)):
        ref, size = rotary_ref(g, inv, pos, layout, mag, -1.0)
        within(got, ref, rotary_tol(ref, size, F32, 1e3), "gradient")
    # the map is linear: <g, rotary(v)> = <grad, v> (fp32 values, summed in 64 bits: 16 U of the absolute terms)
    v = rnd(B, T, H, D, seed=5)
    lhs = (gq.double() * Fn.rotary(v, None, inv, pos, layout=layout, magnitude=mag).double()).sum()
    assert abs(lhs - (dq.double() * v.double()).sum()) <= 32 * U * 2 * (gq.double().abs() * v.double().abs().amax()).sum()
    only = torch.autograd.grad(ko, k, gk, retain_graph=True)[0]
    assert torch.equal(only, dk)
    # keys shared by heads: the heads' gradients add up
    kk = k.detach().clone().requires_grad_()
    out = Fn.rotary(q.detach(), kk.expand(B, T, 4, D), inv, pos, layout=layout, magnitude=mag)[1]
    d = torch.autograd.grad(out, kk, gk.expand(B, T, 4, D))[0]
    within(d, 4 * dk.double(), 4 * 4 * U * dk.abs().double() + 1e-30, "shared")


def test_rotary_nothing_to_do_and_masked_values():
    inv = Fn.rotary_frequencies(8, device="cuda")[0]
    assert Fn.rotary(torch.zeros(0, 3, 2, 8, device="cuda"), None, inv).shape == (0, 3, 2, 8)
    assert Fn.rotary(torch.zeros(2, 0, 2, 8, device="cuda"), torch.zeros(2, 0, 1, 8, device="cuda"), inv)[1].shape == (2, 0, 1, 8)
    x = rnd(1, 4, 2, 8, seed=1)
    want = Fn.rotary(x, None, inv)
    x[0, 2, 1, 3] = float("nan")
    got = Fn.rotary(x, None, inv)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 2, 1, 3] = bad[0, 2, 1, 7] = True        # the value and its partner
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])


def test_rows_past_four_gigabytes():
    """Rows so far apart that their distances from the first pass 32 bits, in elements and in bytes."""
    far = torch.zeros(5 * 2 ** 30, dtype=torch.uint8, device="cuda")
    qa, qb = operands(16500, 2304, 512)
    a = far.view(K.FP8).as_strided((16500, 512), (320000, 1))      # large tiles by its shape: more than their 32 bits reach
    a.copy_(qa[0])
    assert torch.equal(K.gemm_fp8(a, qa[1], *qb), K.gemm_fp8(*qa, *qb))
    qa, qb = operands(3, 40, 256)
    a = far.view(K.FP8).as_strided((3, 256), (2 ** 31 + 16, 1))
    a.copy_(qa[0])
    assert torch.equal(K.gemm_fp8(a, qa[1], *qb), K.gemm_fp8(*qa, *qb))
    x, w = rnd(3, 768, seed=1, dtype=BF16), torch.ones(768, device="cuda")
    xf = far.view(BF16).as_strided((3, 768), (2 ** 30 + 7, 1))
    xf.copy_(x)
    assert torch.equal(K.rms_norm_fwd(xf, w, xf)[0], K.rms_norm_fwd(x, w, x)[0])
    assert torch.equal(K.quant_rows_fp8(xf)[0].view(torch.uint8), K.quant_rows_fp8(x)[0].view(torch.uint8))
    inv = Fn.rotary_frequencies(64, device="cuda")[0]
    t = rnd(3, 2, 4, 64, seed=2, dtype=BF16)
    tf = far.view(BF16).as_strided((3, 2, 4, 64), (2 ** 30, 2 ** 28, 64, 1))
    tf.copy_(t)
    want = Fn.rotary(t, None, inv)
    assert torch.equal(Fn.rotary(tf, None, inv), want)
    Fn.rotary_(tf, None, inv)
    assert torch.equal(tf, want)


def test_a_product_whose_output_passes_four_gigabytes():
    """Rows past the large kernel's 32-bit reach go in launches of their own (small integers: every order of the sums is exact)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    M, N, Kp = 950001, 2304, 256
    ints = [torch.randint(-2, 3, (n, Kp), generator=g, device="cuda", dtype=torch.int8).to(F32).to(K.FP8) for n in (M, N)]
    sa, sb = (torch.full((n, 4), 127, dtype=torch.uint8, device="cuda").view(K.SCALE)[:, :2] for n in (M, N // 128))
    out = K.gemm_fp8(ints[0], sa, ints[1], sb)
    assert out.numel() * 2 > 1 << 32
    w = ints[1].float().t().contiguous()
    for r in (0, 474500, 475136, 949000):
        assert torch.equal(out[r:r + 1001], (ints[0][r:r + 1001].float() @ w).to(BF16)), r
    for r in range(0, M, 100000):      # every row against calls that one launch covers
        assert torch.equal(out[r:r + 100000], K.gemm_fp8(ints[0][r:r + 100000], sa[r:r + 100000], ints[1], sb)), r


def test_rotary_of_more_tokens_than_one_launch_takes():
    T, D = (1 << 23) + 700, 512
    q = rnd(1, 1, 1, D, dtype=BF16).expand(1, T, 1, D)
    inv, _ = Fn.rotary_frequencies(D, device="cuda")
    out = Fn.rotary(q, None, inv)
    for t in (0, 4096, (1 << 23) - 200, T - 300):
        assert torch.equal(out[:, t:t + 300], Fn.rotary(q[:, :300], None, inv, offset=t)), t


# ----------------------------------------------------------------------------------------------------- together, and around
def test_the_chain_into_attention():
    """Norm with residual -> 8-bit projection -> rotary in place on the packed queries and keys -> the framework's attention."""
    B, T, H, D = 3, 65, 12, 768
    M = B * T
    branch, stream = rnd(M, D, seed=1, dtype=BF16), rnd(M, D, seed=2)
    w, wq, bias = 1 + 0.2 * rnd(D, seed=3), torch.nn.Parameter(rnd(3 * D, D, seed=4, scale=0.04)), 0.1 * rnd(3 * D, seed=5)
    inv = Fn.rotary_frequencies(64, device="cuda")[0]
    pos = torch.arange(T, device="cuda") * 2000 + torch.tensor([[0], [90_000_000], [240_000_000]], device="cuda")
    with torch.no_grad():
        q, s, h = Fn.rms_norm_fp8(branch, w, residual=stream)
        qkv = Fn.linear_fp8((q, s), wq, bias)
        packed = qkv.clone().view(B, T, 3 * H, 64)
        Fn.rotary_(packed[:, :, :2 * H], None, inv, pos)
        out, _ = K.attention_fwd(packed.view(M, 3 * D), B, T, H, 64 ** -0.5)
    # every stage against 64 bits on the stage's own input (each bound as in its own test)
    rh, _, ry = norm_ref(branch, w, stream, 1e-6)
    within(h, rh, rh.abs() * U, "h")
    ref, size = product_ref((q, s), Fn.w_fp8(wq), bias)
    within(qkv, ref, ref.abs() * HALF[BF16] + size * PRODUCT_REL + bias.abs().double() * U, "projection")
    ref, size = rotary_ref(qkv.view(B, T, 3 * H, 64)[:, :, :2 * H], inv, pos, "half")
    within(packed[:, :, :2 * H], ref, rotary_tol(ref, size, BF16, 2.5e8), "rotary")
    t = packed.double().view(B, T, 3, H, 64).permute(2, 0, 3, 1, 4)
    p = torch.softmax(torch.matmul(t[0], t[1].transpose(-1, -2).contiguous()) / 8, -1)
    att = torch.matmul(p, t[2].contiguous()).permute(0, 2, 1, 3).reshape(M, D)
    # probabilities and the output are rounded to bf16: 2^-8 each of sum p |v|
    bound = torch.matmul(p, t[2].abs().contiguous()).permute(0, 2, 1, 3).reshape(M, D)
    within(out, att, 3 * HALF[BF16] * bound, "attention")
    # and the whole against the chain in 64 bits without any rounding: 8-bit operands are off by at most 2^-4 each, at random, so the
    # projection's relative error stays below 2^-4 (two operands, each 2^-4 / sqrt(3) rms at the very most)
    whole = torch.mm(ry, wq.detach().double().t().contiguous()) + bias.double()
    assert ((qkv.double() - whole).norm() / whole.norm()).item() < 2.0 ** -4


def test_training_chain_through_attention():
    """Rotary between the projection and the framework's attention, with its gradient: the packed gradient turned back."""
    B, T, H = 2, 65, 2
    D = 64 * H
    inv = Fn.rotary_frequencies(64, device="cuda")[0]
    pos = torch.arange(T, device="cuda") * 3
    qkv, dout = rnd(B * T, 3 * D, seed=1, dtype=BF16), rnd(B * T, D, seed=2, dtype=BF16)
    packed = qkv.clone()
    view = packed.view(B, T, 3 * H, 64)
    K.rotary(view[:, :, :2 * H], None, inv, pos, inplace=True)
    out, lse = K.attention_fwd(packed, B, T, H, 0.125)
    d = K.attention_bwd(packed, out, dout, lse, B, T, H, 0.125)
    K.rotary(d.view(B, T, 3 * H, 64)[:, :, :2 * H], None, inv, pos, backward=True, inplace=True)
    x = qkv.double().requires_grad_()
    t = x.view(B, T, 3 * H, 64)
    turned = torch.cat((rotary_ref(t[:, :, :2 * H], inv, pos, "half")[0], t[:, :, 2 * H:]), 2).view(B, T, 3, H, 64).permute(2, 0, 3, 1, 4)
    p = torch.softmax((turned[0][..., :, None, :] * turned[1][..., None, :, :]).sum(-1) / 8, -1)
    att = (p[..., None] * turned[2][..., None, :, :]).sum(-2).permute(0, 2, 1, 3).reshape(B * T, D)
    want = torch.autograd.grad(att, x, dout.double())[0]
    # six bf16 roundings on the way (rotated q and k, P, dS, output, gradient): relative to the whole, below 6 * 2^-8
    assert ((d.double() - want).norm() / want.norm()).item() < 6 * HALF[BF16]


def test_streams_and_graphs():
    """The same results on another stream and in a graph that is captured once and replayed on new values between eager calls."""
    M, D, N = 37, 768, 256
    x, res, w = rnd(M, D, seed=1, dtype=BF16), rnd(M, D, seed=2), 1 + 0.1 * rnd(D, seed=3)
    wn = torch.nn.Parameter(rnd(N, D, seed=4, scale=0.1))
    fresh = torch.nn.Parameter(wn.detach().clone())                   # has no 8-bit copy when the capture begins
    inv = Fn.rotary_frequencies(64, device="cuda")[0]
    pos = torch.arange(M, device="cuda")

    def chain(x, res, wn):
        with torch.no_grad():
            q, s, h = Fn.rms_norm_fp8(x, w, residual=res)
            y = Fn.linear_fp8((q, s), wn)
            z = Fn.rotary(y.view(1, M, 4, 64), None, inv, pos)
            return q, s, h, y, z, Fn.linear_fp8(res, wn)

    def same(a, b):
        return all(torch.equal(u.view(torch.uint8) if u.element_size() == 1 else u, v.view(torch.uint8) if v.element_size() == 1 else v)
                   for u, v in zip(a, b))
    want = chain(x, res, wn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = chain(x, res, wn)
    torch.cuda.current_stream().wait_stream(side)
    assert same(want, there)
    sx, sres = x.clone(), res.clone()
    graphs = []
    for weight in (wn, fresh):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(sx, sres, weight)
        graphs.append((g, out))
    assert Fn.WEIGHTS.current(fresh, "fp8") is None                   # a copy made inside a capture is not kept
    for i in range(4):
        sx.copy_(rnd(M, D, seed=20 + i, dtype=BF16))
        sres.copy_(rnd(M, D, seed=30 + i))
        eager = chain(sx, sres, wn)
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert same(eager, out), i
    # the training form: forward and backward inside one graph
    tx, tw, tres = x.clone().requires_grad_(), w.clone().requires_grad_(), res.clone().requires_grad_()
    dy, dh = rnd(M, D, seed=5, dtype=BF16), rnd(M, D, seed=6)

    def step():
        y, h = Fn.rms_norm(tx, tw, tres)
        return (y.detach(), h.detach()) + torch.autograd.grad((y, h), (tx, tw, tres), (dy, dh))
    want = [t.clone() for t in step()]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        with torch.no_grad():
            tx.copy_(rnd(M, D, seed=40 + i, dtype=BF16))
        want = [t.clone() for t in step()]


def test_the_same_call_twice_is_the_same():
    """Fixed orders of summation: bit for bit, also for the weight gradient over many rows."""
    x, res, w = rnd(5000, 768, seed=1, dtype=BF16).requires_grad_(), rnd(5000, 768, seed=2).requires_grad_(), torch.ones(768, device="cuda", requires_grad=True)
    dy, dh = rnd(5000, 768, seed=3, dtype=BF16), rnd(5000, 768, seed=4)
    a, b = (torch.autograd.grad(Fn.rms_norm(x, w, res), (x, w, res), (dy, dh)) for _ in range(2))
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    qa, qb = operands(3, 300, 8192)
    assert torch.equal(K.gemm_fp8(*qa, *qb), K.gemm_fp8(*qa, *qb))


def test_one_tensor_in_two_places():
    """The same tensor as input and residual, as both operands' leaves; gradients that share no memory."""
    w = 1 + 0.1 * rnd(96, seed=1)
    x = rnd(5, 96, seed=2).requires_grad_()
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    dy, dh = rnd(5, 96, seed=3), rnd(5, 96, seed=4)
    torch.autograd.backward(Fn.rms_norm(x, w, x, out_dtype=F32), (dy, dh))
    torch.autograd.backward(Fn.rms_norm(a, w, b, out_dtype=F32), (dy, dh))
    assert torch.equal(a.grad, b.grad) and torch.equal(x.grad, a.grad + b.grad)
    a.grad.add_(1)
    assert not torch.equal(a.grad, b.grad)
    # twice through the same weight: its gradient is the sum
    wl = w.clone().requires_grad_()
    y1, y2 = Fn.rms_norm(a.detach(), wl, out_dtype=F32), Fn.rms_norm(dh, wl, out_dtype=F32)
    one, two = (torch.autograd.grad(y, wl, dy, retain_graph=True)[0] for y in (y1, y2))
    assert torch.equal(torch.autograd.grad((y1, y2), wl, (dy, dy))[0], one + two)
    q = rnd(1, 4, 2, 8, seed=5).requires_grad_()
    inv = Fn.rotary_frequencies(8, device="cuda")[0]
    g = rnd(1, 4, 2, 8, seed=6)
    both = torch.autograd.grad(Fn.rotary(q, q, inv), q, (g, g))[0]
    assert torch.equal(both, 2 * torch.autograd.grad(Fn.rotary(q, None, inv), q, g)[0])
    # one buffer as both operands, one row of scales for all rows
    e = K.quant_blocks_fp8(rnd(128, 256, seed=7))
    gram = K.gemm_fp8(e[0], e[1].expand(128, 2), *e)
    assert torch.equal(gram, gram.t())


def test_values_that_a_graph_saved_are_not_overwritten_in_silence():
    x = rnd(1, 4, 2, 8, seed=1)
    w = rnd(1, 4, 2, 8, seed=2).requires_grad_()
    out = (x * w).sum()                     # saves x
    with torch.no_grad():
        Fn.rotary_(x, None, Fn.rotary_frequencies(8, device="cuda")[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()
    with torch.inference_mode():
        t = torch.ones(1, 4, 2, 8, device="cuda")
        Fn.rotary_(t, None, Fn.rotary_frequencies(8, device="cuda")[0])


def test_no_second_derivative_in_silence():
    """A backward pass that is itself to be differentiated is refused: its gradients would be constants."""
    x, w = rnd(4, 96, seed=1).requires_grad_(), torch.ones(96, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(Fn.rms_norm(x, w, out_dtype=F32).sum(), x, create_graph=True)
    q = rnd(1, 3, 2, 8, seed=2).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(Fn.rotary(q, None, Fn.rotary_frequencies(8, device="cuda")[0]).square().sum(), q, create_graph=True)
