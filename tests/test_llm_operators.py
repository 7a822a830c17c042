"""CPU: what the RMS norm, the 8-bit products and the rotary positions refuse, the C entries' own checks, and the rotary frequencies."""
import math

import pytest
import torch

from get_model_amd import functional as Fn
from get_model_amd import kernels as K
from get_model_amd import lib

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: K.rms_norm_fwd(z(4, 8), z(7)),                                             # weight of another width
    lambda: K.rms_norm_fwd(z(4, 8), z(8, dtype=BF16)),                                 # weight type
    lambda: K.rms_norm_fwd(z(4, 8, dtype=torch.float16), z(8)),                        # x type
    lambda: K.rms_norm_fwd(z(4, 8), z(8), z(4, 9)),                                    # residual shape
    lambda: K.rms_norm_fwd(z(4, 8), z(8), z(4, 8, dtype=BF16)),                        # bf16 residual under an fp32 x
    lambda: K.rms_norm_fwd(z(4, 8), z(8), out_dtype=torch.float16),
    lambda: K.rms_norm_fwd(z(4, 8), z(8), eps=-1.0),
    lambda: K.rms_norm_fwd(z(4, 8), z(8), eps=float("nan")),
    lambda: K.rms_norm_fwd(z(8, 4).t(), z(8)),                                         # columns apart
    lambda: K.rms_norm_fwd(z(2, 16385), z(16385)),                                     # too wide
    lambda: K.rms_norm_fwd(z(2, 0), z(0)),
    lambda: K.rms_norm_fp8(z(4, 8), z(8), z(5, 8)),
    lambda: K.rms_norm_bwd(z(4, 8), z(4, 8), z(5), z(8)),
    lambda: K.rms_norm_bwd(z(4, 8), z(4, 8, dtype=BF16), z(4), z(8), bf16_copy=True),
    lambda: K.rms_norm_bwd(z(4, 8), z(4, 8), z(4), z(8), dh=z(4, 8, dtype=BF16)),
    lambda: K.quant_rows_fp8(z(4, 8, 2)),
    lambda: K.quant_rows_fp8(z(4, 8, dtype=torch.float16)),
    lambda: K.quant_rows_fp8(z(1, 16385)),
    lambda: K.quant_blocks_fp8(z(4, 8, dtype=torch.int32)),
    lambda: Fn.rms_norm(z(2, 3, 8), z(8), residual=z(3, 8)),
    lambda: Fn.rms_norm_fp8(z(2, 3, 8), z(8), residual=z(2, 3, 9)),
    lambda: Fn.linear_fp8(z(3, 8), z(5, 9)),
])
def test_norm_and_quantisation_refuse(call):
    with pytest.raises(ValueError):
        call()


def fp8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(K.FP8)


def scales(rows, kb, pitch=None):
    pitch = (kb + 3) // 4 * 4 if pitch is None else pitch
    return torch.full((rows, pitch), 127, dtype=torch.uint8).view(K.SCALE)[:, :kb]


@pytest.mark.parametrize("call", [
    lambda: K.gemm_fp8(fp8(4, 128), scales(4, 1), fp8(8, 256), scales(1, 2)),          # depths differ
    lambda: K.gemm_fp8(fp8(4, 96), scales(4, 1), fp8(8, 96), scales(1, 1)),            # not whole blocks
    lambda: K.gemm_fp8(fp8(4, 128).view(torch.int8), scales(4, 1), fp8(8, 128), scales(1, 1)),
    lambda: K.gemm_fp8(fp8(4, 128), z(4, 1), fp8(8, 128), scales(1, 1)),               # scales in fp32
    lambda: K.gemm_fp8(fp8(4, 128), scales(5, 1), fp8(8, 128), scales(1, 1)),
    lambda: K.gemm_fp8(fp8(4, 128), scales(4, 1), fp8(129, 128), scales(1, 1)),        # two blocks of rows
    lambda: K.gemm_fp8(fp8(4, 128), scales(4, 1, pitch=1), fp8(8, 128), scales(1, 1)),     # scale rows off 4-byte words
    lambda: K.gemm_fp8(fp8(4, 128), torch.full((32,), 127, dtype=torch.uint8).view(K.SCALE)[1:].as_strided((4, 1), (4, 1), 1),
                       fp8(8, 128), scales(1, 1)),                                     # ... all of them
    lambda: K.gemm_fp8(fp8(4, 136)[:, :128], scales(4, 1), fp8(8, 128), scales(1, 1)),     # rows off 16 bytes
    lambda: K.gemm_fp8(fp8(4, 128), scales(4, 1), fp8(8, 128), scales(1, 1), bias=z(7)),
    lambda: K.gemm_fp8(fp8(4, 128), scales(4, 1), fp8(8, 128), scales(1, 1), bias=z(8, dtype=BF16)),
    lambda: K.linear_rows_fp8(z(17, 100), fp8(8, 128), scales(1, 1)),                  # too many rows
    lambda: K.linear_rows_fp8(z(4, 200), fp8(8, 128), scales(1, 1)),                   # deeper than the weight
    lambda: K.linear_rows_fp8(z(4, 100, dtype=torch.float16), fp8(8, 128), scales(1, 1)),
    lambda: K.linear_rows_fp8(z(4, 100), fp8(8, 128), scales(1, 1), bias=z(7)),
])
def test_products_refuse(call):
    with pytest.raises(ValueError):
        call()


INV = Fn.rotary_frequencies(8)[0]
X = z(2, 3, 6, 8)


@pytest.mark.parametrize("call", [
    lambda: K.rotary(z(2, 3, 8), None, INV),                                           # three dimensions
    lambda: K.rotary(z(2, 3, 4, 6), None, INV),                                        # narrower than the rotated columns
    lambda: K.rotary(z(2, 3, 4, 8), None, INV.float()),
    lambda: K.rotary(z(2, 3, 4, 8), None, INV[:0]),
    lambda: K.rotary(z(2, 3, 4, 8), z(2, 4, 4, 8), INV),                               # k of another length
    lambda: K.rotary(z(2, 3, 4, 8), z(2, 3, 4, 8, dtype=BF16), INV),
    lambda: K.rotary(z(2, 3, 4, 8, dtype=torch.float16), None, INV),
    lambda: K.rotary(z(2, 3, 4, 8), None, INV, positions=z(3)),                        # positions in fp32
    lambda: K.rotary(z(2, 3, 4, 8), None, INV, positions=torch.arange(4)),
    lambda: K.rotary(z(2, 3, 4, 8), None, INV, positions=torch.arange(3), offset=1),
    lambda: K.rotary(z(2, 3, 4, 8), None, INV, layout="pairs"),
    lambda: K.rotary(z(2, 3, 8, 4).transpose(2, 3), None, INV),                        # columns apart
    lambda: K.rotary(z(2, 3, 1, 8).expand(2, 3, 4, 8), None, INV, inplace=True),       # elements share memory
    lambda: K.rotary(z(1, 1, 1, 4098), None, torch.ones(1025, dtype=F64)),
    lambda: K.rotary(z(1, 1, 1, 8), None, INV, offset=2 ** 53),
    lambda: K.rotary(X, X, INV, inplace=True),                                         # q and k the same, shifted, interleaved
    lambda: K.rotary(X[:, :-1], X[:, 1:], INV, inplace=True),
    lambda: K.rotary(X[:, :, :4], X[:, :, 3:], INV, inplace=True),
    lambda: K.rotary(X[..., 0:8], X.view(2, 3, 48)[:, :, 4:44].unflatten(2, (5, 8)), INV, inplace=True),
])
def test_rotary_refuses(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("Hq,Hk", [(4, 2), (1, 5), (3, 3), (6, 0)])
def test_parts_of_one_layout_do_not_share(Hq, Hk):
    """Queries and keys of a packed projection, in either order, heads before or behind the tokens: exactly the calls that touch no
    element twice pass (the rule against a count of every element)."""
    B, T, D = 2, 3, 8
    H = Hq + Hk + 1
    for buf in (torch.arange(B * T * H * D).view(B, T, H, D), torch.arange(B * H * T * D).view(B, H, T, D).transpose(1, 2),
                torch.arange(T * B * H * D).view(T, B, H, D).transpose(0, 1)):
        for a in range(H - Hq + 1):
            for b in range(H - Hk + 1):
                q, k = buf[:, :, a:a + Hq], buf[:, :, b:b + Hk]
                both = torch.cat((q.reshape(-1), k.reshape(-1)))
                assert K._share(q, k) == (both.unique().numel() < both.numel()), (a, b)
    rows = torch.arange(B * (T + 1) * H * D).view(B, T + 1, H, D)
    if Hk:
        assert K._share(rows[:, :T, :Hk], rows[:, 1:, :Hk])


def test_no_cpu_fallback():
    for call in (lambda: K.rms_norm_fwd(z(4, 8), z(8)), lambda: K.rms_norm_fp8(z(4, 8), z(8)), lambda: K.quant_rows_fp8(z(4, 8)),
                 lambda: K.quant_blocks_fp8(z(4, 8)), lambda: K.rotary(z(2, 3, 4, 8), None, INV), lambda: Fn.linear_fp8(z(3, 8), z(5, 8)),
                 lambda: K.gemm_fp8(fp8(4, 128), scales(4, 1), fp8(8, 128), scales(1, 1)), lambda: Fn.rms_norm(z(4, 8), z(8))):
        with pytest.raises(RuntimeError):
            call()


def test_inference_operators_refuse_gradients():
    w = torch.nn.Parameter(z(8))
    with pytest.raises(RuntimeError, match="no_grad"):
        Fn.rms_norm_fp8(z(4, 8), w)
    with pytest.raises(RuntimeError, match="no_grad"):
        Fn.linear_fp8(z(4, 8), torch.nn.Parameter(z(8, 8)))
    with pytest.raises(RuntimeError, match="no_grad"):
        Fn.rotary_(z(1, 1, 1, 8).requires_grad_(), None, INV)


def test_c_entries_check_before_they_launch():
    """Bad sizes and null pointers come back as error 1 with a message; nothing is launched (there is no GPU here)."""
    h, p, n = lib.load(), 4096, None
    bad = [
        ("getmi_rmsnorm_fwd", (p, 0, 8, n, 0, 0, p, p, 0, n, n, 4, 0, 1e-6, n)),       # no columns
        ("getmi_rmsnorm_fwd", (p, 0, 8, n, 0, 0, p, p, 0, n, n, 4, 20000, 1e-6, n)),   # too wide
        ("getmi_rmsnorm_fwd", (n, 0, 8, n, 0, 0, p, p, 0, n, n, 4, 8, 1e-6, n)),       # no x
        ("getmi_rmsnorm_fwd", (p, 0, 8, p, 0, 8, p, p, 0, n, n, 4, 8, 1e-6, n)),       # residual without h
        ("getmi_rmsnorm_fwd", (p, 2, 8, n, 0, 0, p, p, 0, n, n, 4, 8, 1e-6, n)),       # unknown type
        ("getmi_rmsnorm_fp8", (p, 0, 8, n, 0, 0, p, p, p, 0, n, 4, 8, 1e-6, n)),       # scale rows too short
        ("getmi_rmsnorm_fp8", (p, 0, 8, p, 0, 8, n, p, p, 4, p, 4, 8, 1e-6, n)),       # residual without a norm
        ("getmi_rmsnorm_bwd", (p, 0, p, 0, 8, p, p, n, p, n, p, 4, 8, n, 0, n)),       # dw without workspace
        ("getmi_rmsnorm_bwd", (p, 0, p, 1, 8, p, p, n, p, p, n, 4, 8, n, 0, n)),       # bf16 copy next to bf16
        ("getmi_quant_blocks_fp8", (p, 0, 8, p, p, 0, 8, 8, n)),
        ("getmi_gemm_fp8", (p, p, p, p, n, p, 4, 4, 100, 128, 128, 4, 4, 4, n, 0, n)),       # depth not whole blocks
        ("getmi_gemm_fp8", (p, p, p, p, n, p, 4, 4, 128, 120, 128, 4, 4, 4, n, 0, n)),       # rows off 16 bytes
        ("getmi_gemm_fp8", (p, p, p, p, n, p, 4, 4, 128, 128, 128, 3, 4, 4, n, 0, n)),       # output rows overlap
        ("getmi_gemm_fp8", (p, p, p, p, n, p, 4, 4, 128, 128, 128, 4, 5, 4, n, 0, n)),       # scale rows off 4 bytes
        ("getmi_gemm_fp8", (p, p, p, p, n, p, 64, 64, 8192, 8192, 8192, 64, 64, 64, n, 0, n)),     # split depth without workspace
        ("getmi_linear_fp8_rows", (p, 0, 128, p, p, n, p, 17, 64, 128, 128, 64, 4, n)),            # too many rows
        ("getmi_linear_fp8_rows", (p, 2, 128, p, p, n, p, 4, 64, 128, 128, 64, 4, n)),             # unknown type
        ("getmi_linear_fp8_rows", (p, 0, 128, p, p, n, p, 4, 64, 128, 100, 64, 4, n)),             # rows off 16 bytes
        ("getmi_rotary", (p, p, 1, n, n, 0, n, 0, 1, 1, 8, 8, p, n, 0, 0, 0, 0, 0, 0, 1.0, n)),      # no strides
        ("getmi_rotary", (p, p, 1, n, n, 0, p, 0, 1, 1, 8, 7, p, n, 0, 0, 0, 0, 0, 0, 1.0, n)),      # odd columns
        ("getmi_rotary", (p, p, 1, n, n, 0, p, 0, 1, 1, 8, 16, p, n, 0, 0, 0, 0, 0, 0, 1.0, n)),     # more than the head has
    ]
    for name, args in bad:
        assert getattr(h, name)(*args) == 1, (name, args)
        assert h.getmi_last_error()
    # nothing to do is no error
    assert h.getmi_rmsnorm_fwd(n, 0, 8, n, 0, 0, n, n, 0, n, n, 0, 8, 1e-6, n) == 0
    assert h.getmi_gemm_fp8(n, n, n, n, n, n, 0, 4, 128, 128, 128, 4, 4, 4, n, 0, n) == 0
    assert h.getmi_rotary(n, n, 0, n, n, 0, n, 0, 1, 1, 8, 8, n, n, 0, 0, 0, 0, 0, 0, 1.0, n) == 0


def test_linear_in_tiles_checks_before_it_launches():
    h, p, n = lib.load(), 4096, None
    for args in [(p, 0, 128, p, p, n, p, -1, 64, 128, 128, 64, 4, n),       # rows
                 (p, 2, 128, p, p, n, p, 17, 64, 128, 128, 64, 4, n),       # unknown type
                 (p, 0, 128, p, p, n, p, 17, 64, 128, 100, 64, 4, n),       # weight rows off 16 bytes
                 (p, 0, 128, p, p, n, p, 17, 64, 128, 128, 63, 4, n),       # output rows overlap
                 (p, 0, 128, p, p, n, p, 17, 64, 128, 128, 64, 5, n),       # scale rows off 4 bytes
                 (n, 0, 128, p, p, n, p, 17, 64, 128, 128, 64, 4, n)]:      # no x
        assert h.getmi_linear_fp8_tiles(*args) == 1 and h.getmi_last_error(), args
    assert h.getmi_linear_fp8_tiles(n, 0, 0, n, n, n, n, 0, 64, 128, 128, 64, 4, n) == 0
    w = torch.zeros(64, 128).to(K.FP8), torch.zeros(1, 4, dtype=torch.uint8).view(K.SCALE)[:, :1]
    for x in (torch.zeros(20, 128, dtype=F64), torch.zeros(20, 129), torch.zeros(128), torch.zeros(20, 16385)):
        with pytest.raises(ValueError):
            K.linear_tiles_fp8(x, *w)
    with pytest.raises(RuntimeError):      # no CPU path
        K.linear_tiles_fp8(torch.zeros(20, 128), *w)


def test_c_entries_refuse_more_than_a_launch_holds():
    h, p, n, most = lib.load(), 4096, None, 0x7fff0000
    assert h.getmi_gemm_fp8(p, p, p, p, n, p, most, 64, 128, 128, 128, 64, 4, 4, n, 0, n) == 1
    assert b"too large" in h.getmi_last_error()
    assert h.getmi_linear_fp8_rows(p, 0, 128, p, p, n, p, 4, most, 128, 128, most, 4, n) == 1
    assert b"too large" in h.getmi_last_error()


def test_rotary_frequencies():
    c, base = 64, 10000.0
    plain, m = Fn.rotary_frequencies(c, base)
    want = torch.tensor([base ** (-2 * i / c) for i in range(c // 2)], dtype=F64)
    assert plain.dtype == F64 and m == 1.0 and torch.allclose(plain, want, rtol=1e-15, atol=0)
    linear, m = Fn.rotary_frequencies(c, base, "linear", 8.0)
    assert m == 1.0 and torch.equal(linear, plain / 8)
    ntk, m = Fn.rotary_frequencies(c, base, "ntk", 8.0)
    # the highest frequency stays, the lowest is divided by the factor, all fall in between
    assert m == 1.0 and ntk[0] == plain[0] and math.isclose(ntk[-1], plain[-1] / 8, rel_tol=1e-12) and bool((ntk <= plain).all())
    yarn, m = Fn.rotary_frequencies(c, base, "yarn", 8.0, original_length=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(m, 0.1 * math.log(8) + 1)
    assert torch.equal(yarn[turns > 40], plain[turns > 40]) and torch.equal(yarn[turns < 0.8], plain[turns < 0.8] / 8)
    mid = (turns < 30) & (turns > 1.2)
    assert mid.any() and bool((yarn[mid] < plain[mid]).all()) and bool((yarn[mid] > plain[mid] / 8).all())
    for bad in (dict(columns=7), dict(columns=0), dict(columns=8, factor=0.5), dict(columns=8, scaling="cubic"), dict(columns=8, base=0.0),
                dict(columns=8, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            Fn.rotary_frequencies(**bad)
