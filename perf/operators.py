"""The cases on which the large-model operators are measured: the root-mean-square norm with the residual's addition (training
form, and the serving form that leaves 8-bit values with scales), the 8-bit block-scaled product that consumes those values, and
rotary positions on queries and keys.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, where the module's `own` is true, with the
framework's kernels; `exact` computes it in 64 bits from the operator's definition.  Sizes: the training batch of the benchmark
(256 samples of 200 regions and a CLS token, embed_dim 768, 12 heads of 64), its parts, and generic ones.

Definitions (row r, block = 128 consecutive columns, rounded to the output's type once at the end)
  norm      h = x + residual;  y = w * h / sqrt(mean(h^2) + eps)
  backward  dh' = dh + rstd * (w*dy - hhat * mean(w*dy*hhat)), hhat = h*rstd;  dx = dresidual = dh';  dw = sum_rows dy*hhat
  8 bits    per block: scale = the smallest power of two with max|y| <= 448 * scale (1 for an all-zero block), q = e4m3(y / scale);
            rows are padded with zeros to whole blocks
  product   out (bf16) = sum_b sa[m,b] * sb[n/128,b] * sum_{k in b} qa[m,k]*qb[n,k]  (+ bias)
  rotary    pair (u, v) at angle a = position * inv_freq:  (u cos a - v sin a, v cos a + u sin a) * magnitude; pairs are (i, i + R/2)
            ("half") or (2i, 2i+1) ("interleaved") of the first R columns of a head, the others pass through
"""
import math

import torch

own = False

EPS = 1e-6
BLOCK = 128
E4M3_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4, "none": 0}


def listed():
    norm = dict(op="norm_train")
    fp8 = dict(op="norm_fp8")
    mm = dict(op="product")
    rot = dict(op="rotary")
    return [
        # one encoder block's norm in the training step: a bf16 branch output added to the fp32 residual stream, and its backward
        dict(norm, name="norm train, whole batch", M=51456, D=768, x="bf16", res="f32", out="bf16"),
        # a narrow odd-width feature table (283 motif columns), a few samples, no residual
        dict(norm, name="norm train, odd width", M=804, D=283, x="f32", res="none", out="f32"),
        # serving one new token: a launch's latency
        dict(fp8, name="norm to 8 bits, one token", M=1, D=768, x="bf16", res="f32"),
        # serving a whole batch: the norm in front of the 8-bit projections
        dict(fp8, name="norm to 8 bits, whole batch", M=51456, D=768, x="bf16", res="f32"),
        # one token through a wide projection: the weights' bytes are the time
        dict(mm, name="product, one token", M=1, N=8192, K=8192, bias=False),
        # one sample (200 regions and CLS) through the packed query-key-value projection
        dict(mm, name="product, one sample", M=201, N=2304, K=768, bias=True),
        # the whole batch through the same projection
        dict(mm, name="product, whole batch", M=51456, N=2304, K=768, bias=True),
        # a large square product: the matrix units' rate
        dict(mm, name="product, large", M=8192, N=8192, K=8192, bias=False),
        # a projection whose input is still in 16 bits (the attention's output): quantised and multiplied in one call
        dict(op="linear", name="linear from 16 bits", M=4020, N=768, K=768, bias=True),
        # decoding: one token for each of 64 sequences, every one at a position of its own
        dict(rot, name="rotary, one token each", B=64, T=1, Hq=12, Hk=12, D=64, R=64, layout="half", x="bf16", positions="offsets",
             train=False, stretch=1.0),
        # training: queries and keys inside the packed projection, positions are base pairs on a chromosome; with gradients
        dict(rot, name="rotary train, base pairs", B=256, T=201, Hq=12, Hk=12, D=64, R=64, layout="half", x="bf16",
             positions="genomic", train=True, stretch=1.0),
        # a long context, stretched eightfold: half of each head rotated, interleaved, few key heads
        dict(rot, name="rotary, long context", B=1, T=32768, Hq=16, Hk=2, D=128, R=64, layout="interleaved", x="f32",
             positions="index", train=False, stretch=8.0),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_train", "norm_fp8", "product", "product", "linear", "rotary", "rotary"])
    if op in ("norm_train", "norm_fp8"):
        D = _spread(rng, 33, 8192)
        M = _spread(rng, 1, max(2, min(51456, 51456 * 768 // D)))
        x = rng.choice(["bf16", "f32"])
        res = rng.choice(["none", "f32"]) if x == "f32" else rng.choice(["none", "f32", "bf16"])
        c = dict(op=op, M=M, D=D, x=x, res=res)
        if op == "norm_train":
            c["out"] = rng.choice(["bf16", "f32"])
        return c
    if op in ("product", "linear"):
        N, K = _spread(rng, 17, 8192), _spread(rng, 65, 8192)
        M = _spread(rng, 1, max(2, min(51456, (1 << 38) // (N * K), (1 << 27) // N, (1 << 27) // K)))
        return dict(op=op, M=M, N=N, K=K, bias=rng.random() < 0.5)
    D = 2 * _spread(rng, 8, 128)
    R = D if rng.random() < 0.5 else 2 * rng.randint(2, D // 2)
    Hq = _spread(rng, 1, 64)
    Hk = rng.choice([Hq, max(1, Hq // 4), 1])
    tokens = _spread(rng, 1, max(2, min(131072, 51456 * 1536 // ((Hq + Hk) * D))))
    T = 1 if rng.random() < 0.25 else _spread(rng, 1, tokens)
    return dict(op="rotary", B=max(1, tokens // T), T=T, Hq=Hq, Hk=Hk, D=D, R=R, layout=rng.choice(["half", "interleaved"]),
                x=rng.choice(["bf16", "f32"]), positions=rng.choice(["offsets", "genomic", "index"]), train=rng.random() < 0.4,
                stretch=rng.choice([1.0, 1.0, 4.0, 16.0]))


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _activations(g, M, D, dtype):
    """Rows as a deep encoder's residual stream has them: of unlike size, with a few large columns."""
    t = torch.randn(M, D, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(M, 1, generator=g, device="cuda"))
    return (t * torch.exp(0.7 * torch.randn(1, D, generator=g, device="cuda"))).to(dtype)


def _power(e):
    """2^e as float32 for int32 exponents of normal numbers."""
    return ((e + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e (448 = 0.875 * 2^9; frexp's fraction is in [0.5, 1)); 0 for amax = 0."""
    m, e = torch.frexp(amax)
    e = e.to(torch.int32) - 9 + (m > 0.875).to(torch.int32)
    return torch.where(amax == 0, torch.zeros_like(e), e.clamp(min=-126))


def _padded(v, rows=1):
    """v[R, K] with zeros up to whole multiples of `rows` and of the block."""
    R, K = v.shape
    return torch.nn.functional.pad(v, (0, -K % BLOCK, 0, -R % rows))


def _scales(e):
    """Scale bytes (exponent + 127) as an 8-bit exponent tensor whose rows start on 4-byte words."""
    R, Kb = e.shape
    t = torch.full((R, (Kb + 3) // 4 * 4), 127, dtype=torch.uint8, device=e.device)
    t[:, :Kb] = (e + 127).to(torch.uint8)
    return t.view(torch.float8_e8m0fnu)[:, :Kb]


def _quant_rows(v):
    """float32 [R, K] -> (e4m3 [R, Kp], scales [R, Kp/128]): one scale for each row and block."""
    p = _padded(v)
    b = p.view(p.shape[0], -1, BLOCK)
    e = _exponent(b.abs().amax(-1))
    return (b * _power(-e)[..., None]).view(p.shape).to(torch.float8_e4m3fn), _scales(e)


def _quant_weight(w):
    """float32 [N, K] -> (e4m3 [N, Kp], scales [ceil(N/128), Kp/128]): one scale for each 128 x 128 block."""
    N = w.shape[0]
    p = _padded(w, BLOCK)
    b = p.view(p.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    e = _exponent(b.abs().amax((1, 3)))
    q = (b * _power(-e)[:, None, :, None]).view(p.shape)[:N].to(torch.float8_e4m3fn)
    return q.contiguous(), _scales(e)


def _inv_freq(c):
    """Frequencies of a context stretched by `stretch` through a larger base (angles are formed in 64 bits)."""
    R = c["R"]
    base = 10000.0 * c["stretch"] ** (R / max(R - 2, 1))
    return base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)


def prepare(case, seed):
    c, g = case, _generator(seed)
    if c["op"] in ("norm_train", "norm_fp8"):
        M, D = c["M"], c["D"]
        s = dict(case=c, x=_activations(g, M, D, TYPES[c["x"]]), w=1.0 + 0.2 * _randn(g, D), res=None)
        if c["res"] != "none":
            s["res"] = _activations(g, M, D, TYPES[c["res"]])
        if c["op"] == "norm_train":
            s["dy"] = _randn(g, M, D, dtype=TYPES[c["out"]])
            s["dh"] = None if s["res"] is None else _randn(g, M, D, dtype=TYPES[c["res"]])
            for k in ("x", "res", "w"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    if c["op"] in ("product", "linear"):
        M, N, K = c["M"], c["N"], c["K"]
        s = dict(case=c, b=_quant_weight(0.05 * _randn(g, N, K)), bias=_randn(g, N) if c["bias"] else None)
        x = _activations(g, M, K, torch.bfloat16)
        s["x"] = x if c["op"] == "linear" else _quant_rows(x.float())
        return s
    B, T, D, x = c["B"], c["T"], c["D"], TYPES[c["x"]]
    # queries and keys lie in one packed projection, next to the values
    packed = _randn(g, B, T, c["Hq"] + 2 * c["Hk"], D, dtype=x)
    s = dict(case=c, q=packed[:, :, :c["Hq"]], k=packed[:, :, c["Hq"]:c["Hq"] + c["Hk"]], inv_freq=_inv_freq(c).cuda(),
             magnitude=0.1 * math.log(c["stretch"]) + 1.0)
    start = torch.randint(0, 230_000_000 if c["positions"] == "genomic" else 100_000, (B, 1), generator=g, device="cuda")
    if c["positions"] == "genomic":      # peaks some two thousand base pairs apart
        gap = (-2000.0 * torch.rand(B, T, generator=g, device="cuda").clamp(min=1e-6).log()).long() + 200
        s["positions"] = start + gap.cumsum(1)
    elif c["positions"] == "offsets":
        s["positions"] = start + torch.arange(T, device="cuda")
    else:
        s["positions"] = torch.arange(T, device="cuda")
    if c["train"]:
        s["q"], s["k"] = s["q"].requires_grad_(), s["k"].requires_grad_()
        s["gq"], s["gk"] = _randn(g, B, T, c["Hq"], D, dtype=x), _randn(g, B, T, c["Hk"], D, dtype=x)
    return s


# ------------------------------------------------------------------------------------------------------------------- run
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from get_model_amd import functional as Fn
    c = s["case"]
    if c["op"] == "norm_train":
        out_type = TYPES[c["out"]]
        if s["res"] is None:
            y = Fn.rms_norm(s["x"], s["w"], eps=EPS, out_dtype=out_type)
            return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        y, h = Fn.rms_norm(s["x"], s["w"], residual=s["res"], eps=EPS, out_dtype=out_type)
        return (y.detach(), h.detach()) + torch.autograd.grad((y, h), (s["x"], s["w"], s["res"]), (s["dy"], s["dh"]))
    if c["op"] == "norm_fp8":
        return Fn.rms_norm_fp8(s["x"], s["w"], residual=s["res"], eps=EPS)
    if c["op"] in ("product", "linear"):
        return Fn.linear_fp8(s["x"], s["b"], bias=s["bias"])
    kw = dict(positions=s["positions"], layout=c["layout"], magnitude=s["magnitude"])
    q, k = Fn.rotary(s["q"], s["k"], s["inv_freq"], **kw)
    if not c["train"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))


def _turn(x, cos, sin, c):
    """The rotation of x[B,T,H,D] by angles whose cosines and sines are [.., T, 1, R/2]."""
    R, t = c["R"], x.float()
    if c["layout"] == "half":
        u, v = t[..., :R // 2], t[..., R // 2:R]
        out = torch.cat((u * cos - v * sin, v * cos + u * sin), -1)
    else:
        u, v = t[..., 0:R:2], t[..., 1:R:2]
        out = torch.stack((u * cos - v * sin, v * cos + u * sin), -1).flatten(-2)
    return torch.cat((out, t[..., R:]), -1).to(x.dtype)


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    if c["op"] in ("norm_train", "norm_fp8"):
        x, w, res = s["x"], s["w"], s["res"]
        h = x.float() if res is None else x.float() + res.float()
        rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        y = h * rstd * w
        if c["op"] == "norm_fp8":
            return _quant_rows(y) if res is None else _quant_rows(y) + (h.to(res.dtype),)
        hhat, dy = h * rstd, s["dy"].float()
        dn = dy * w
        d = rstd * (dn - hhat * (dn * hhat).mean(-1, keepdim=True))
        dw = (dy * hhat).sum(0, dtype=torch.float64).float()
        y = y.to(TYPES[c["out"]])
        if res is None:
            return y, d.to(x.dtype), dw
        d = d + s["dh"].float()
        return y, h.to(res.dtype), d.to(x.dtype), dw, d.to(res.dtype)
    if c["op"] in ("product", "linear"):
        a, sa = s["x"] if c["op"] == "product" else _quant_rows(s["x"].float())
        b, sb = s["b"]
        fa = _power(sa.view(torch.uint8).int() - 127).repeat_interleave(BLOCK, 1)
        fb = _power(sb.view(torch.uint8).int() - 127).repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 0)[:b.shape[0]]
        out = (a.float() * fa) @ (b.float() * fb).t()
        return (out if s["bias"] is None else out + s["bias"]).to(torch.bfloat16)
    a = s["positions"].double()[..., None] * s["inv_freq"]
    cos, sin = ((f(a) * s["magnitude"]).float().unsqueeze(-2) for f in (torch.cos, torch.sin))
    q, k = _turn(s["q"], cos, sin, c), _turn(s["k"], cos, sin, c)
    if not c["train"]:
        return q, k
    return q, k, _turn(s["gq"], cos, -sin, c), _turn(s["gk"], cos, -sin, c)


# ----------------------------------------------------------------------------------------------------------- definitions
def work(case):
    c = case
    if c["op"] == "norm_train":
        M, D, x, r, o = c["M"], c["D"], SIZE[c["x"]], SIZE[c["res"]], SIZE[c["out"]]
        # x, residual, dy, dh in; y, h, dx, dresidual out; the weight and its gradient
        return {"bytes": M * D * (2 * x + 4 * r + 2 * o) + 8 * D, "flops": 14.0 * M * D}
    if c["op"] == "norm_fp8":
        M, D = c["M"], c["D"]
        return {"bytes": M * D * (SIZE[c["x"]] + 2 * SIZE[c["res"]] + 1) + M * -(-D // BLOCK) + 4 * D, "flops": 7.0 * M * D}
    if c["op"] in ("product", "linear"):
        M, N, K = c["M"], c["N"], c["K"]
        a = M * K * 2 if c["op"] == "linear" else M * K + M * -(-K // BLOCK)
        return {"bytes": a + N * K + -(-N // BLOCK) * -(-K // BLOCK) + M * N * 2 + (4 * N if c["bias"] else 0),
                "flops": 2.0 * M * N * K}
    n = c["B"] * c["T"] * (c["Hq"] + c["Hk"]) * c["D"] * (2 if c["train"] else 1)
    return {"bytes": 2 * n * SIZE[c["x"]] + 8 * c["T"] * (1 if c["positions"] == "index" else c["B"]) + 4 * c["R"], "flops": 3.0 * n}


def _exact_blocks(v, rows):
    """64-bit v[R, K] -> (v / scale, scale) over blocks of `rows` x 128, v padded to whole blocks in K."""
    R, K = v.shape
    Rb, Kb = -(-R // rows), -(-K // BLOCK)
    full = v.new_zeros(Rb * rows, Kb * BLOCK)
    full[:R, :K] = v
    full = full.reshape(Rb, rows, Kb, BLOCK)
    most = full.abs().amax((1, 3), keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(most / E4M3_MAX)))
    scale = torch.where(most / scale > E4M3_MAX, scale * 2, torch.where(most / scale <= E4M3_MAX / 2, scale / 2, scale))
    scale = torch.where(most == 0, torch.ones_like(scale), scale)
    return (full / scale).reshape(Rb * rows, Kb * BLOCK)[:R], scale.reshape(Rb, Kb)


def _to_e4m3(v):
    """The e4m3 values nearest to v (ties to even): 4 significant bits, the smallest step 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    with torch.no_grad():
        s, c = prepare(case, seed), case
        if c["op"] in ("norm_train", "norm_fp8"):
            h = s["x"].double()
            if s["res"] is not None:
                h = h + s["res"].double()
            w, D = s["w"].double(), h.shape[1]
            root = (h.pow(2).sum(1, keepdim=True) / D + EPS).sqrt()
            n = h / root
            if c["op"] == "norm_fp8":
                q, scale = _exact_blocks(n * w, 1)
                return (q, scale) if s["res"] is None else (q, scale, h)
            dy = s["dy"].double()
            dh = (dy * w - n * ((dy * w * n).sum(1, keepdim=True) / D)) / root
            if s["res"] is None:
                return n * w, dh, (dy * n).sum(0)
            dh = dh + s["dh"].double()
            return n * w, h, dh, (dy * n).sum(0), dh
        if c["op"] in ("product", "linear"):
            if c["op"] == "product":
                a, e = s["x"][0].double(), s["x"][1].view(torch.uint8).double() - 127
            else:
                a, scale = _exact_blocks(s["x"].double(), 1)
                a, e = _to_e4m3(a), torch.log2(scale)
            b, f = s["b"][0].double(), s["b"][1].view(torch.uint8).double() - 127
            M, N = a.shape[0], b.shape[0]
            a = (a.reshape(M, -1, BLOCK) * torch.exp2(e)[:, :, None]).reshape(M, -1)
            f = torch.exp2(f)[torch.arange(N, device=b.device) // BLOCK]
            b = (b.reshape(N, -1, BLOCK) * f[:, :, None]).reshape(N, -1)
            out = torch.mm(a, b.t().contiguous())
            return out if s["bias"] is None else out + s["bias"].double()
        angle = (s["positions"].double().reshape(-1, c["T"], 1) * s["inv_freq"]).expand(c["B"], -1, -1)[:, :, None]
        z = torch.polar(torch.full_like(angle, s["magnitude"]), angle)
        R = c["R"]

        def turned(x, z):
            x = x.double()
            if c["layout"] == "half":
                y = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * z
                y = torch.cat((y.real, y.imag), -1)
            else:
                y = torch.view_as_real(torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], R // 2, 2)) * z).flatten(-2)
            return torch.cat((y, x[..., R:]), -1)

        q, k = turned(s["q"], z), turned(s["k"], z)
        return (q, k, turned(s["gq"], z.conj()), turned(s["gk"], z.conj())) if c["train"] else (q, k)
