"""Tensor-level wrappers of the C-ABI kernels (one Python function per entry point of include/getmi355.h).

torch is used only to allocate device buffers and to provide the stream; all arithmetic happens in
libgetmi355.so.  Every function requires CUDA(HIP) tensors and raises RuntimeError otherwise.
"""
import ctypes
import functools

import torch

from . import lib

EPI_BF16, EPI_BIAS_GELU, EPI_BIAS_RESID, EPI_DGELU, EPI_EMBED, EPI_F32, EPI_BIAS_GELUG, EPI_DMUL = range(8)
BF16 = torch.bfloat16
F32 = torch.float32

# bench.py sets PROFILE = [] to collect (kernel name, algorithmic flops, start event, end event) per GEMM launch,
# recorded on the stream the kernel is launched on (torch's current stream).
PROFILE = None
# when a set: only these kernel groups get events (an event pair per launch keeps consecutive kernels from overlapping
# their ramp-up / tail: ~0.9 ms per C2 step with every GEMM and attention launch bracketed, ~0.2 ms with one group)
PROFILE_ONLY = None
_EPI_NAMES = ("bf16", "bias_gelu", "bias_resid", "dgelu", "embed", "f32", "bias_gelu", "dgelu")   # 6, 7: training forms


def _prof_begin(name):
    if PROFILE is None or (PROFILE_ONLY is not None and name not in PROFILE_ONLY):
        return None
    e = torch.cuda.Event(enable_timing=True)
    e.record()
    return e


def _prof_end(e0, name, flops):
    if e0 is None:
        return
    e1 = torch.cuda.Event(enable_timing=True)
    e1.record()
    PROFILE.append((name, flops, e0, e1))


def _chk(*ts):
    for t in ts:
        if t is not None and not (t.is_cuda and t.is_contiguous()):
            raise RuntimeError("getmi355 kernels need contiguous tensors on the GPU (no CPU fallback exists)")


def _ws(nbytes, device):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def cast_pad(src, cp=None):
    """fp32 [R,C] -> bf16 [R,Cp] (zero padded)."""
    _chk(src)
    R, C = src.shape
    cp = C if cp is None else cp
    dst = torch.empty(R, cp, dtype=BF16, device=src.device)
    lib.call("getmi_cast_pad_f32_bf16", src, dst, R, C, cp)
    return dst


def cast_bf16(src):
    """fp32 tensor -> bf16 tensor of the same shape (numel % 4 == 0)."""
    _chk(src)
    n = src.numel()
    dst = torch.empty(src.shape, dtype=BF16, device=src.device)
    lib.call("getmi_cast_pad_f32_bf16", src, dst, 1, n, n)
    return dst


def cast_transpose(src):
    """fp32 [R,C] -> bf16 [C,R]."""
    _chk(src)
    R, C = src.shape
    dst = torch.empty(C, R, dtype=BF16, device=src.device)
    lib.call("getmi_cast_transpose_f32_bf16", src, dst, R, C)
    return dst


def qkv_bias(q_bias, v_bias):
    _chk(q_bias, v_bias)
    D = q_bias.numel()
    out = torch.empty(3 * D, dtype=F32, device=q_bias.device)
    lib.call("getmi_qkv_bias", q_bias, v_bias, out, D)
    return out


def gemm_tn(epi, A, B, out0, out1=None, bias=None, resid=None, rowscale=None, rows_per_sample=0, aux=None,
            mask=None, mask_token=None, regions_per_sample=0, M=None, dbias=None, prescaled=False, blocked=False):
    """out = epilogue(A[M,K] @ B[N,K]^T).  A, B bf16 row-major; out0/out1 preallocated (out0 may be None for the
    two-output GELU epilogues: only gelu(u) is stored).  blocked: out0 of EPI_BIAS_GELUG / aux of EPI_DMUL is a
    `blocked_rows(M)` x N buffer in the hand-over layout of getmi355.h (flags bit 1; ask gemm_tn_blocked_ok first)."""
    _chk(A, B, out0, out1, bias, resid, rowscale, aux, mask, mask_token)
    M = A.shape[0] if M is None else M
    K = A.shape[1]
    N = B.shape[0]
    assert B.shape[1] == K and A.dtype == BF16 and B.dtype == BF16
    ws = None if dbias is None else _ws(lib.query("getmi_gemm_tn_workspace_bytes", M, N), A.device)
    e0 = _prof_begin("gemm_tn_kernel<" + _EPI_NAMES[epi] + ">")
    ldo = (out0 if out0 is not None else out1).shape[-1]
    lib.call("getmi_gemm_tn", epi, A, B, M, N, K, A.stride(0), B.stride(0), out0, out1, ldo, bias,
             resid, rowscale, rows_per_sample, aux, 0 if aux is None else aux.shape[-1], mask, mask_token,
             regions_per_sample, dbias, ws, 0 if ws is None else ws.numel(), (1 if prescaled else 0) | (2 if blocked else 0))
    _prof_end(e0, "gemm_tn_kernel<" + _EPI_NAMES[epi] + ">", 2.0 * M * N * K)
    return out0


def gemm_tn_blocked_ok(M, N, K):
    """May fc1's forward hand gelu'(u) to fc2's data gradient in the blocked layout (same answer for both calls)?"""
    return bool(lib.query("getmi_gemm_tn_blocked_ok", M, N, K))


def blocked_rows(M):
    return (M + 15) // 16 * 16


def gemm_wgrad(X, Y, out=None, accumulate=False):
    """out[N1,N2] (+)= X[M,N1]^T @ Y[M,N2]  (fp32)."""
    _chk(X, Y, out)
    M, N1 = X.shape
    N2 = Y.shape[1]
    assert Y.shape[0] == M and X.dtype == BF16 and Y.dtype == BF16
    if out is None:
        out = torch.empty(N1, N2, dtype=F32, device=X.device)
        accumulate = False
    nbytes = lib.query("getmi_gemm_wgrad_workspace_bytes", M, N1, N2)
    ws = _ws(nbytes, X.device)
    e0 = _prof_begin("gemm_wgrad_kernel(+reduce_slabs)")
    lib.call("getmi_gemm_wgrad", X, Y, M, N1, N2, X.stride(0), Y.stride(0), out, int(accumulate), ws, ws.numel())
    _prof_end(e0, "gemm_wgrad_kernel(+reduce_slabs)", 2.0 * M * N1 * N2)
    return out


def gemm_wgrad_pair(Xa, Ya, Xb, Yb, out_a=None, out_b=None):
    """(Xa^T @ Ya, Xb^T @ Yb) for operands with the same number of rows, in one launch."""
    _chk(Xa, Ya, Xb, Yb, out_a, out_b)
    M = Xa.shape[0]
    assert Ya.shape[0] == M and Xb.shape[0] == M and Yb.shape[0] == M
    N1a, N2a, N1b, N2b = Xa.shape[1], Ya.shape[1], Xb.shape[1], Yb.shape[1]
    if out_a is None:
        out_a = torch.empty(N1a, N2a, dtype=F32, device=Xa.device)
    if out_b is None:
        out_b = torch.empty(N1b, N2b, dtype=F32, device=Xa.device)
    ws = _ws(lib.query("getmi_gemm_wgrad_pair_workspace_bytes", M, N1a, N2a, N1b, N2b), Xa.device)
    e0 = _prof_begin("gemm_wgrad_kernel(+reduce_slabs)")
    lib.call("getmi_gemm_wgrad_pair", Xa, Ya, N1a, N2a, Xa.stride(0), Ya.stride(0), out_a, 0, Xb, Yb, N1b, N2b, Xb.stride(0),
             Yb.stride(0), out_b, 0, M, ws, ws.numel())
    _prof_end(e0, "gemm_wgrad_kernel(+reduce_slabs)", 2.0 * M * (N1a * N2a + N1b * N2b))
    return out_a, out_b


def layernorm_fwd(x, gamma, beta, eps=1e-6):
    """x fp32 [M,D] -> (y bf16 [M,D], mean [M], rstd [M])."""
    _chk(x, gamma, beta)
    M, D = x.shape
    y = torch.empty(M, D, dtype=BF16, device=x.device)
    mean = torch.empty(M, dtype=F32, device=x.device)
    rstd = torch.empty(M, dtype=F32, device=x.device)
    e0 = _prof_begin("ln_fwd_kernel")
    lib.call("getmi_layernorm_fwd", x, gamma, beta, y, mean, rstd, M, D, float(eps))
    _prof_end(e0, "ln_fwd_kernel", float(M) * D * 6)         # algorithmic bytes: x fp32 in, y bf16 out
    return y, mean, rstd


def layernorm_bwd(dy, x, mean, rstd, gamma, dres=None, rowscale=None, rows_per_sample=0, want_dz=False,
                  want_dbias=False, dx_dtype=F32):
    """Returns (dx, dz bf16|None, dgamma, dbeta, dbias_prev|None).  dres may be fp32 or bf16; dx_dtype picks the element
    type of dx (the "bf16 gradient stream" of functional.py passes bf16 on both sides).  With a bf16 dx and no row scale
    dz IS dx (same tensor: the kernel does not write it twice)."""
    _chk(dy, x, mean, rstd, gamma, dres, rowscale)
    M, D = x.shape
    dev = x.device
    dx = torch.empty(M, D, dtype=dx_dtype, device=dev)
    alias = want_dz and dx_dtype == BF16 and rowscale is None
    dz = torch.empty(M, D, dtype=BF16, device=dev) if (want_dz and not alias) else None
    dgamma = torch.empty(D, dtype=F32, device=dev)
    dbeta = torch.empty(D, dtype=F32, device=dev)
    dbias = torch.empty(D, dtype=F32, device=dev) if want_dbias else None
    ws = _ws(lib.query("getmi_layernorm_bwd_workspace_bytes", M, D), dev)
    e0 = _prof_begin("ln_bwd_kernel")
    res_b = dres is not None and dres.dtype == BF16
    if res_b or dx_dtype == BF16:
        lib.call("getmi_layernorm_bwd_stream", dy, x, mean, rstd, gamma, dres, int(res_b), rowscale, rows_per_sample, dx,
                 int(dx_dtype == BF16), dz, dgamma, dbeta, dbias, 0, M, D, ws, ws.numel())
    else:
        lib.call("getmi_layernorm_bwd", dy, x, mean, rstd, gamma, dres, rowscale, rows_per_sample, dx, dz, dgamma, dbeta,
                 dbias, 0, M, D, ws, ws.numel())
    # (for this HBM-bound kernel the profile's second field is its ALGORITHMIC BYTES, not FLOPs: dy bf16 + x fp32 +
    #  dx (+ dres) in their stream type (+ dz bf16) per element)
    sb = 2 if dx_dtype == BF16 else 4
    rb = 0 if dres is None else (2 if res_b else 4)
    _prof_end(e0, "ln_bwd_kernel", float(M) * D * (2 + 4 + sb + rb + (2 if dz is not None else 0)))
    return dx, (dx if alias else dz), dgamma, dbeta, dbias


def attention_fwd(qkv, B, T, H, scale, want_lo=False, sample_scale=None):
    """qkv bf16 [B*T, 3*H*64] (packed [B,T,3,H,64]) -> (out bf16 [B*T, H*64], lse fp32 [B,H,T]); with want_lo also
    the rounding residual bf16(O - out) that attention_bwd takes as out_lo."""
    _chk(qkv, sample_scale)
    out = torch.empty(B * T, H * 64, dtype=BF16, device=qkv.device)
    lo = torch.empty(B * T, H * 64, dtype=BF16, device=qkv.device) if want_lo else None
    lse = torch.empty(B, H, T, dtype=F32, device=qkv.device)
    e0 = _prof_begin("attn_fwd_kernel")
    lib.call("getmi_attention_fwd", qkv, out, lo, lse, B, T, H, float(scale), sample_scale)
    _prof_end(e0, "attn_fwd_kernel", 4.0 * B * H * T * T * 64)
    return (out, lse, lo) if want_lo else (out, lse)


def attention_bwd(qkv, out, dout, lse, B, T, H, scale, want_bias=False, out_lo=None, sample_scale=None):
    """-> dqkv, or (dqkv, dq_bias [H*64], dv_bias [H*64]) with want_bias (column sums of the Q / V thirds, fp32)."""
    _chk(qkv, out, dout, lse, out_lo, sample_scale)
    dqkv = torch.empty_like(qkv)
    dqb = torch.empty(H * 64, dtype=F32, device=qkv.device) if want_bias else None
    dvb = torch.empty(H * 64, dtype=F32, device=qkv.device) if want_bias else None
    ws = _ws(lib.query("getmi_attention_bwd_workspace_bytes", B, T, H), qkv.device)
    e0 = _prof_begin("attn_bwd_kernel(+delta)")
    lib.call("getmi_attention_bwd", qkv, out, out_lo, dout, lse, dqkv, dqb, dvb, B, T, H, float(scale), sample_scale, ws,
             ws.numel())
    _prof_end(e0, "attn_bwd_kernel(+delta)", 10.0 * B * H * T * T * 64)
    return (dqkv, dqb, dvb) if want_bias else dqkv


def fill_cls(x0, cls_token, B, T, D):
    _chk(x0, cls_token)
    lib.call("getmi_fill_cls", x0, cls_token, B, T, D)


def embed_bwd_prep(dx0, mask_u8, B, N, D):
    """-> (dz bf16 [B*N,D], dcls [D], dmask_token [D], dbias [D])."""
    _chk(dx0, mask_u8)
    dev = dx0.device
    dz = torch.empty(B * N, D, dtype=BF16, device=dev)
    dcls = torch.empty(D, dtype=F32, device=dev)
    dmt = torch.empty(D, dtype=F32, device=dev)
    dbias = torch.empty(D, dtype=F32, device=dev)
    ws = _ws(lib.query("getmi_embed_bwd_workspace_bytes", B, N, D), dev)
    lib.call("getmi_embed_bwd_prep", dx0, mask_u8, dz, dcls, dmt, dbias, 0, B, N, D, ws, ws.numel())
    return dz, dcls, dmt, dbias


def head_fwd(hf, W, bias, B, N):
    _chk(hf, W, bias)
    out_dim, D = W.shape
    logits = torch.empty(B, N, out_dim, dtype=F32, device=hf.device)
    pred = torch.empty(B, N, out_dim, dtype=F32, device=hf.device)
    lib.call("getmi_head_fwd", hf, W, bias, logits, pred, B, N, D, out_dim)
    return logits, pred


def head_bwd(dpred, logits, hf, W, B, N):
    """-> (dh bf16 [B*(N+1), D], dW [out,D], db [out])."""
    _chk(dpred, logits, hf, W)
    out_dim, D = W.shape
    dev = hf.device
    dh = torch.empty(B * (N + 1), D, dtype=BF16, device=dev)
    dwb = torch.empty(out_dim * D + out_dim, dtype=F32, device=dev)
    ws = _ws(lib.query("getmi_head_bwd_workspace_bytes", B, N, D, out_dim), dev)
    lib.call("getmi_head_bwd", dpred, logits, hf, W, dh, dwb, 0, B, N, D, out_dim, ws, ws.numel())
    return dh, dwb[: out_dim * D].view(out_dim, D), dwb[out_dim * D:]


LOSS_POISSON, LOSS_MSE = 0, 1


def loss_fwd(kind, pred, obs, weight=1.0, eps=1e-8):
    """pred/obs: 2-D views [R, C] with unit column stride -> (loss scalar tensor, grad_unit like pred)."""
    assert pred.dim() == 2 and obs.dim() == 2 and pred.stride(1) == 1 and obs.stride(1) == 1
    if not (pred.is_cuda and obs.is_cuda):
        raise RuntimeError("getmi355 kernels need GPU tensors")
    R, C = pred.shape
    loss = torch.empty((), dtype=F32, device=pred.device)
    grad = torch.empty(R, C, dtype=F32, device=pred.device)
    ws = _ws(lib.query("getmi_loss_workspace_bytes"), pred.device)
    lib.call("getmi_loss_fwd", kind, pred, obs, loss, grad, R, C, pred.stride(0), obs.stride(0), C, float(weight),
             float(eps), ws, ws.numel())
    return loss, grad


def scale_by_scalar(x, scalar, weight=1.0):
    _chk(x, scalar)
    out = torch.empty_like(x)
    lib.call("getmi_scale_by_scalar", x, scalar, float(weight), out, x.numel())
    return out


def scale_cast(dx, rowscale=None, rows_per_sample=0):
    """dx fp32 [M,D] -> (dz bf16 = rowscale*dx, dbias [D] = column sums of dz)."""
    _chk(dx, rowscale)
    M, D = dx.shape
    dz = torch.empty(M, D, dtype=BF16, device=dx.device)
    dbias = torch.empty(D, dtype=F32, device=dx.device)
    ws = _ws(lib.query("getmi_scale_cast_workspace_bytes", M, D), dx.device)
    lib.call("getmi_scale_cast", dx, rowscale, rows_per_sample, dz, dbias, 0, M, D, ws, ws.numel())
    return dz, dbias


def gather_rows(src, idx, n_out=None, scatter=False):
    """gather: dst[i] = src[idx[i]]; scatter: dst[idx[i]] = src[i] (dst zero-initialised, n_out rows)."""
    _chk(src, idx)
    D = src.shape[1]
    n = idx.numel()
    if scatter:
        dst = torch.zeros(n_out, D, dtype=BF16, device=src.device)
    else:
        dst = torch.empty(n, D, dtype=BF16, device=src.device)
    lib.call("getmi_gather_rows_bf16", src, idx, dst, n, D, int(scatter))
    return dst


def mask_compact(mask_u8, B, N):
    """mask uint8 [B*N] -> (token_rows int64 [B*N], region_rows int64 [B*N], count int32 [1]); only the first
    count[0] entries of the row lists are defined.  No host synchronisation."""
    _chk(mask_u8)
    dev = mask_u8.device
    tok = torch.empty(B * N, dtype=torch.int64, device=dev)
    reg = torch.empty(B * N, dtype=torch.int64, device=dev)
    cnt = torch.empty(1, dtype=torch.int32, device=dev)
    lib.call("getmi_mask_compact", mask_u8, B, N, tok, reg, cnt)
    return tok, reg, cnt


def colsum_bf16(X, M=None):
    """Column sums of a bf16 matrix (row stride may exceed the column count: column slices are fine)."""
    if not (X.is_cuda and X.stride(1) == 1):
        raise RuntimeError("getmi355 kernels need GPU tensors with unit column stride")
    M = X.shape[0] if M is None else M
    N = X.shape[1]
    out = torch.empty(N, dtype=F32, device=X.device)
    ws = _ws(lib.query("getmi_colsum_workspace_bytes", N), X.device)
    lib.call("getmi_colsum_bf16", X, out, 0, M, N, X.stride(0), ws, ws.numel())
    return out


def scale_cast_noalloc(dx, rowscale=None, rows_per_sample=0):
    """scale_cast through the entry point that uses the library's built-in scratch buffer (no workspace argument; for
    callers that cannot allocate).  The two result tensors here are the caller's outputs, as in the C ABI."""
    _chk(dx, rowscale)
    M, D = dx.shape
    dz = torch.empty(M, D, dtype=BF16, device=dx.device)
    dbias = torch.empty(D, dtype=F32, device=dx.device)
    lib.call("getmi_scale_cast_noalloc", dx, rowscale, rows_per_sample, dz, dbias, 0, M, D)
    return dz, dbias


# ---- root-mean-square norm, 8-bit block-scaled products, rotary positions ---------------------------------------------------
# These check shapes and types first (ValueError, also for CPU tensors), then that every tensor is on one GPU (RuntimeError),
# and run on the tensors' own GPU whatever the current one is.  One token's call is bound by this Python: no message is formatted
# and no object made before a check fails.
FP8 = torch.float8_e4m3fn
SCALE = torch.float8_e8m0fnu        # 2^(byte - 127)
FP8_BLOCK = 128
_TYPE = {F32: 0, BF16: 1}
_MOST = 0x7fff0000                  # rows / tokens: the kernels step past the end in 32 bits


def _refuse(what):
    raise ValueError("getmi355: " + what)


def _on_gpu(*ts):
    """The one GPU of all tensors (None is skipped)."""
    index = dev = None
    for t in ts:
        if t is not None:
            i = t.get_device()
            if i != index:
                if i < 0:
                    raise RuntimeError("getmi355 kernels need tensors on the GPU (no CPU fallback exists)")
                if index is not None:
                    raise RuntimeError(f"getmi355: tensors on two GPUs ({dev} and {t.device})")
                index, dev = i, t.device
    return dev


def _rows(t, what):
    """2-D rows of contiguous columns -> distance of the rows in elements (0 for one row that stands for all)."""
    if t.dim() != 2:
        _refuse(f"{what} has to be 2-D (rows of columns), got {tuple(t.shape)}")
    ld, step = t.stride()
    M, D = t.shape
    if step != 1 and D > 1:
        _refuse(f"the columns of {what} have to be contiguous")
    if M > _MOST or D > _MOST:
        _refuse(f"{what} is too large: {M} x {D}")
    return ld


def _norm_args(x, weight, residual, eps):
    ldx = _rows(x, "x")
    if x.dtype not in _TYPE:
        _refuse(f"x has to be float32 or bfloat16, got {x.dtype}")
    D = x.shape[1]
    if not 0 < D <= 16384:
        _refuse(f"the norm takes 1 to 16384 columns, got {D}")
    if weight.dtype != F32 or weight.shape != (D,) or not weight.is_contiguous():
        _refuse(f"the norm's weight has to be contiguous float32 [{D}], got {weight.dtype} {tuple(weight.shape)}")
    ldr = 0
    if residual is not None:
        if residual.shape != x.shape:
            _refuse(f"residual {tuple(residual.shape)} and x {tuple(x.shape)} differ in shape")
        if residual.dtype != F32 and residual.dtype != x.dtype:
            _refuse(f"the residual has to be float32 or of x's type, got {residual.dtype}")
        ldr = _rows(residual, "the residual")
    if not eps >= 0:
        _refuse(f"eps has to be >= 0, got {eps}")
    return ldx, ldr, D


def rms_norm_fwd(x, weight, residual=None, eps=1e-6, out_dtype=BF16, want_rstd=False):
    """x fp32 / bf16 [M,D] (rows may lie apart), weight fp32 [D] -> (y, h, rstd).  h = x + residual in the residual's type (None
    without a residual), y = weight * h / sqrt(mean(h^2) + eps) in out_dtype, rstd fp32 [M] (None unless wanted)."""
    ldx, ldr, D = _norm_args(x, weight, residual, eps)
    if out_dtype not in _TYPE:
        _refuse(f"out_dtype has to be float32 or bfloat16, got {out_dtype}")
    dev = _on_gpu(x, weight, residual)
    M = x.shape[0]
    y = torch.empty(M, D, dtype=out_dtype, device=dev)
    h = None if residual is None else torch.empty(M, D, dtype=residual.dtype, device=dev)
    rstd = torch.empty(M, dtype=F32, device=dev) if want_rstd else None
    if M:
        lib.launch("getmi_rmsnorm_fwd", dev, x.data_ptr(), _TYPE[x.dtype], ldx, None if residual is None else residual.data_ptr(),
                   0 if residual is None else _TYPE[residual.dtype], ldr, weight.data_ptr(), y.data_ptr(), _TYPE[out_dtype],
                   None if h is None else h.data_ptr(), None if rstd is None else rstd.data_ptr(), M, D, eps)
    return y, h, rstd


def rms_norm_bwd(dy, h, rstd, weight, dh=None, want_dw=True, bf16_copy=False):
    """-> (dx, dx2, dw).  dy fp32 / bf16 [M,D], h [M,D] (what was normalised; rows may lie apart), dh of h's type or None.
    dx in h's type is the gradient of x and of the residual alike; dx2 is dx in bf16 (only with bf16_copy and an fp32 h)."""
    _rows(h, "h")
    M, D = h.shape
    if dy.shape != h.shape or dy.dtype not in _TYPE or not dy.is_contiguous():
        _refuse("dy has to be contiguous float32 or bfloat16 of h's shape")
    if h.dtype not in _TYPE or not 0 < D <= 16384:
        _refuse("h has to be float32 or bfloat16 with 1 to 16384 columns")
    if rstd.shape != (M,) or rstd.dtype != F32 or not rstd.is_contiguous():
        _refuse(f"rstd has to be contiguous float32 [{M}]")
    if weight.dtype != F32 or weight.shape != (D,) or not weight.is_contiguous():
        _refuse(f"weight has to be contiguous float32 [{D}]")
    if dh is not None and (dh.shape != h.shape or dh.dtype != h.dtype or not dh.is_contiguous()):
        _refuse("dh has to be contiguous, of h's shape and type")
    if bf16_copy and h.dtype != F32:
        _refuse("a bf16 copy of dx is made next to an fp32 one only")
    return rms_norm_bwd_unchecked(dy, h, rstd, weight, dh, want_dw, bf16_copy, _on_gpu(dy, h, rstd, weight, dh))


@functools.lru_cache(maxsize=256)
def _rms_norm_bwd_workspace(M, D):
    return max(lib.query("getmi_rmsnorm_bwd_workspace_bytes", M, D), 256)


def rms_norm_bwd_unchecked(dy, h, rstd, weight, dh, want_dw, bf16_copy, dev):
    """rms_norm_bwd for a caller that knows its arguments to be right (functional: what the forward saved, autograd's gradients)."""
    M, D = h.shape
    dx = torch.empty(M, D, dtype=h.dtype, device=dev)
    dx2 = torch.empty(M, D, dtype=BF16, device=dev) if bf16_copy else None
    if M == 0:
        return dx, dx2, torch.zeros(D, dtype=F32, device=dev) if want_dw else None
    dw = ws = None
    need = 0
    if want_dw:
        need = _rms_norm_bwd_workspace(M, D)
        dw = torch.empty(D, dtype=F32, device=dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    lib.launch("getmi_rmsnorm_bwd", dev, dy.data_ptr(), _TYPE[dy.dtype], h.data_ptr(), _TYPE[h.dtype], h.stride(0), rstd.data_ptr(),
               weight.data_ptr(), None if dh is None else dh.data_ptr(), dx.data_ptr(), None if dx2 is None else dx2.data_ptr(),
               None if dw is None else dw.data_ptr(), M, D, None if ws is None else ws.data_ptr(), need)
    return dx, dx2, dw


def _fp8_like(rows, scale_rows, cols, device):
    """Empty values [rows, Kp] and scales [scale_rows, Kp/128] whose rows start on 4-byte words, and the words' bytes a row."""
    kb = -(-cols // FP8_BLOCK)
    pitch = (kb + 3) // 4 * 4
    return (torch.empty(rows, kb * FP8_BLOCK, dtype=FP8, device=device),
            torch.empty_strided((scale_rows, kb), (pitch, 1), dtype=SCALE, device=device), pitch)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """rms_norm_fwd with y left as e4m3 values and power-of-two scales -> (q [M,Kp], scales [M,Kp/128], h)."""
    ldx, ldr, D = _norm_args(x, weight, residual, eps)
    dev = _on_gpu(x, weight, residual)
    M = x.shape[0]
    q, s, pitch = _fp8_like(M, M, D, dev)
    h = None if residual is None else torch.empty(M, D, dtype=residual.dtype, device=dev)
    if M:
        lib.launch("getmi_rmsnorm_fp8", dev, x.data_ptr(), _TYPE[x.dtype], ldx, None if residual is None else residual.data_ptr(),
                   0 if residual is None else _TYPE[residual.dtype], ldr, weight.data_ptr(), q.data_ptr(), s.data_ptr(), pitch,
                   None if h is None else h.data_ptr(), M, D, eps)
    return q, s, h


def quant_rows_fp8(x):
    """x fp32 / bf16 [M,K] -> (q e4m3 [M,Kp], scales [M,Kp/128]): one power-of-two scale per row and 128 columns."""
    ldx = _rows(x, "x")
    M, D = x.shape
    if x.dtype not in _TYPE or not 0 < D <= 16384:
        _refuse(f"quantisation takes float32 or bfloat16 with 1 to 16384 columns, got {x.dtype} [{M}, {D}]")
    dev = _on_gpu(x)
    q, s, pitch = _fp8_like(M, M, D, dev)
    if M:
        lib.launch("getmi_rmsnorm_fp8", dev, x.data_ptr(), _TYPE[x.dtype], ldx, None, 0, 0, None, q.data_ptr(), s.data_ptr(),
                   pitch, None, M, D, 0.0)
    return q, s


def quant_blocks_fp8(w):
    """weight fp32 / bf16 [N,K] -> (q e4m3 [N,Kp], scales [ceil(N/128),Kp/128]): one power-of-two scale per 128 x 128 block."""
    ldw = _rows(w, "the weight")
    N, Kd = w.shape
    if w.dtype not in _TYPE or Kd == 0:
        _refuse(f"quantisation takes float32 or bfloat16 [N,K], got {w.dtype} [{N}, {Kd}]")
    dev = _on_gpu(w)
    q, s, pitch = _fp8_like(N, -(-N // FP8_BLOCK), Kd, dev)
    if N:
        lib.launch("getmi_quant_blocks_fp8", dev, w.data_ptr(), _TYPE[w.dtype], ldw, q.data_ptr(), s.data_ptr(), pitch, N, Kd)
    return q, s


def _fp8_operand(q, s, rows, what):
    """Checks of one operand -> distances of its rows of values and of scales in bytes."""
    if q.dtype != FP8 or s.dtype != SCALE:
        _refuse(f"{what} has to be (float8_e4m3fn, float8_e8m0fnu), got ({q.dtype}, {s.dtype})")
    ld = _rows(q, what)
    lds = _rows(s, "the scales")
    cols = q.shape[1]
    if cols & 127 or cols == 0:
        _refuse(f"{what} has to be padded to whole blocks of 128 columns, got {cols}")
    if s.shape[0] != rows or s.shape[1] != cols >> 7:
        _refuse(f"the scales of {what} have to be [{rows}, {cols >> 7}], got {tuple(s.shape)}")
    if (ld | q.data_ptr()) & 15:
        _refuse(f"the rows of {what} have to start on 16 bytes")
    if rows <= 1:       # a single row's distance means nothing
        lds = 0
    if (lds | s.data_ptr()) & 3 or lds > _MOST:
        _refuse(f"the scale rows of {what} have to start on 4-byte words, less than 2 GiB apart")
    return ld, lds


def gemm_fp8(a, a_scale, b, b_scale, bias=None):
    """bf16 [M,N] = a[M,Kp] @ b[N,Kp]^T (+ bias fp32 [N]) with the scales of quant_rows_fp8 (a) and quant_blocks_fp8 (b)."""
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        _refuse(f"operands {tuple(a.shape)} and {tuple(b.shape)} do not match")
    M, Kp = a.shape
    N = b.shape[0]
    lda, lsa = _fp8_operand(a, a_scale, M, "a")
    ldb, lsb = _fp8_operand(b, b_scale, -(-N // FP8_BLOCK), "b")
    if bias is not None and (bias.dtype != F32 or bias.shape != (N,) or not bias.is_contiguous()):
        _refuse(f"bias has to be contiguous float32 [{N}]")
    dev = _on_gpu(a, a_scale, b, b_scale, bias)
    out = torch.empty(M, N, dtype=BF16, device=dev)
    if M and N:
        ws, need = None, lib.query("getmi_gemm_fp8_workspace_bytes", M, N, Kp) if Kp >= 6144 else 0      # a shallower one is never split
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        lib.launch("getmi_gemm_fp8", dev, a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(),
                   None if bias is None else bias.data_ptr(), out.data_ptr(), M, N, Kp, lda, ldb, N, lsa, lsb,
                   None if ws is None else ws.data_ptr(), need)
    return out


def linear_rows_fp8(x, b, b_scale, bias=None):
    """gemm_fp8 of up to 16 rows x[M,K] in fp32 / bf16, quantised inside the product (bit for bit quant_rows_fp8 + gemm_fp8)."""
    return _linear_inside("getmi_linear_fp8_rows", 16, x, b, b_scale, bias)


def linear_tiles_fp8(x, b, b_scale, bias=None):
    """The same for any number of rows: every 64 x 64 tile quantises the rows it reads, which pays where there are few tiles."""
    return _linear_inside("getmi_linear_fp8_tiles", _MOST, x, b, b_scale, bias)


def _linear_inside(entry, most, x, b, b_scale, bias):
    ldx = _rows(x, "x")
    M, Kd = x.shape
    N = b.shape[0]
    if x.dtype not in _TYPE or not 0 < Kd <= 16384 or M > most:
        _refuse(f"float32 or bfloat16 of at most {most} rows and 16384 columns is wanted, got {x.dtype} [{M}, {Kd}]")
    ldb, lsb = _fp8_operand(b, b_scale, -(-N // FP8_BLOCK), "b")
    if b.shape[1] != -(-Kd // FP8_BLOCK) * FP8_BLOCK:
        _refuse(f"x {tuple(x.shape)} and b {tuple(b.shape)} do not match")
    if bias is not None and (bias.dtype != F32 or bias.shape != (N,) or not bias.is_contiguous()):
        _refuse(f"bias has to be contiguous float32 [{N}]")
    dev = _on_gpu(x, b, b_scale, bias)
    out = torch.empty(M, N, dtype=BF16, device=dev)
    if M and N:
        lib.launch(entry, dev, x.data_ptr(), _TYPE[x.dtype], ldx, b.data_ptr(), b_scale.data_ptr(),
                   None if bias is None else bias.data_ptr(), out.data_ptr(), M, N, Kd, ldb, N, lsb)
    return out


def _overlaps(t):
    """May two elements of t share memory?  (Dimensions in order of stride: each has to step over all the smaller ones.)"""
    end = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st < end:
            return True
        end = st * n
    return False


def _share(q, k):
    """May q[B,T,Hq,D] and k[B,T,Hk,D], neither of which overlaps itself, share elements?  No if their addresses lie apart, or if they
    are parts of one layout: equal strides, and k's start one more step in the order of the strides."""
    if not q.numel() or not k.numel():
        return False
    span = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))) for t in (q, k)]
    if span[0][1] <= span[1][0] or span[1][1] <= span[0][0]:
        return False
    low, high = (q, k) if q.data_ptr() <= k.data_ptr() else (k, q)
    step = (high.data_ptr() - low.data_ptr()) // q.element_size()
    dims = []
    for a, b, st, st2 in zip(low.shape, high.shape, low.stride(), high.stride()):
        if max(a, b) > 1:
            if a > 1 and b > 1 and st != st2:
                return True
            dims.append((st if a > 1 else st2, a, b))
    ends, placed = [1, 1], False
    for st, a, b in sorted(dims):
        if not placed and step < st:
            if step < ends[0]:
                return True
            ends, placed = [step + ends[1]] * 2, True
        if st < max(ends):
            return True
        ends = [st * max(a, b)] * 2 if placed else [st * a, st * b]
    return not placed and step < ends[0]


_Strides = ctypes.c_int64 * 12


def rotary(q, k, inv_freq, positions=None, offset=0, layout="half", magnitude=1.0, backward=False, inplace=False):
    """q [B,T,Hq,D] and k [B,T,Hk,D] (or None), fp32 or bf16, any strides with contiguous columns -> rotated (q, k), new contiguous
    tensors or, inplace, q and k themselves.  inv_freq: float64 [R/2] on the GPU, R <= D rotated columns; positions: int32 / int64
    [B,T] or [T] (None: offset, offset + 1, ..); layout "half" or "interleaved"; backward: by the opposite angle."""
    if q.dim() != 4:
        _refuse(f"q has to be [B, T, heads, D], got {tuple(q.shape)}")
    B, T, Hq, D = q.shape
    dtype = q.dtype
    if dtype not in _TYPE:
        _refuse(f"q has to be float32 or bfloat16, got {dtype}")
    if layout != "half" and layout != "interleaved":
        _refuse(f"layout has to be 'half' or 'interleaved', got {layout!r}")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        _refuse("inv_freq has to be contiguous float64 [R/2]")
    R = 2 * inv_freq.shape[0]
    if not 0 < R <= min(D, 2048):
        _refuse(f"{R} rotated columns do not fit heads of {D} (at most 2048)")
    if q.stride(3) != 1 and D > 1:
        _refuse("the columns of q have to be contiguous")
    Hk = 0
    if k is not None:
        if k.dim() != 4 or k.dtype != dtype or k.shape[0] != B or k.shape[1] != T or k.shape[3] != D:
            _refuse(f"k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {dtype}")
        Hk = k.shape[2]
        if k.stride(3) != 1 and D > 1:
            _refuse("the columns of k have to be contiguous")
    if B * T > _MOST or Hq + Hk > 65536:
        _refuse(f"at most {_MOST} tokens and 65536 heads, got {B * T} and {Hq + Hk}")
    if not -2 ** 53 < offset < 2 ** 53:
        _refuse(f"offset {offset} is not below 2^53")
    if positions is not None:
        if positions.dtype != torch.int64 and positions.dtype != torch.int32:
            _refuse(f"positions have to be int64 or int32, got {positions.dtype}")
        if offset != 0:
            _refuse("positions and an offset exclude each other")
        if positions.shape != (B, T) and positions.shape != (T,):
            _refuse(f"positions have to be [{B}, {T}] or [{T}], got {tuple(positions.shape)}")
    if inplace and (_overlaps(q) or (k is not None and (_overlaps(k) or _share(q, k)))):
        _refuse("in place needs tensors whose elements do not share memory")
    return rotary_unchecked(q, k, inv_freq, positions, offset, layout, magnitude, backward, inplace, _on_gpu(q, k, inv_freq, positions))


def rotary_unchecked(q, k, inv_freq, positions, offset, layout, magnitude, backward, inplace, dev):
    """rotary for a caller that knows its arguments to be right."""
    B, T, Hq, D = q.shape
    qb, qt, qh, _ = q.stride()
    dtype = q.dtype
    Hk = kb = kt = kh = pb = pt = wide = 0
    qo, ko = q, k
    if k is not None:
        Hk = k.shape[2]
        kb, kt, kh, _ = k.stride()
    if positions is not None:
        wide = int(positions.dtype == torch.int64)
        if positions.dim() == 2:
            pb, pt = positions.stride()
        else:
            pt = positions.stride(0)
    if inplace:
        strides = _Strides(qb, qt, qh, qb, qt, qh, kb, kt, kh, kb, kt, kh)
    else:
        qo = torch.empty(B, T, Hq, D, dtype=dtype, device=dev)
        if k is not None:
            ko = torch.empty(B, T, Hk, D, dtype=dtype, device=dev)
        strides = _Strides(qb, qt, qh, T * Hq * D, Hq * D, D, kb, kt, kh, T * Hk * D, Hk * D, D)
    if B * T * (Hq + Hk):
        lib.launch("getmi_rotary", dev, q.data_ptr(), qo.data_ptr(), Hq, None if k is None else k.data_ptr(),
                   None if k is None else ko.data_ptr(), Hk, strides, _TYPE[dtype], B, T, D, 2 * inv_freq.shape[0], inv_freq.data_ptr(),
                   None if positions is None else positions.data_ptr(), wide, pb, pt, offset, layout == "interleaved", backward, magnitude)
    return qo, ko
