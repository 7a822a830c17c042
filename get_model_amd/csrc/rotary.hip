// Rotary positions: pair (u, v) of a head at angle a = position * inv_freq becomes
//     (u cos a - v sin a, v cos a + u sin a) * magnitude          (backward: the same with -a)
// Pairs are (i, i + R/2) ("half") or (2i, 2i + 1) ("interleaved") of the first R columns; columns R .. D-1 pass through.
//
// Positions may be base pairs on a chromosome (2.5e8) or further: the angle is formed and reduced to a quarter turn in 64
// bits (product with its rounding error, two-part pi/2), which leaves |r| <= pi/4 to fp32 polynomials (Taylor, remainder below
// 3e-9 for the sine and 2e-9 for the cosine).  A workgroup forms the R/2 cosines and sines of its few tokens once, in LDS, so
// the 64-bit work is a small fraction and every head reads them back; q and k share one launch.  HBM-bound: every element is
// read once and written once, 16 bytes per lane.
//
// Measured (a 1-GiB copy reaches 5.0 TB/s): 256 x 201 x 24 heads of 64 bf16, half: 63 us (316 MB, 5.0 TB/s), in place 69;
// 32768 x 18 x 128 fp32, interleaved, half of the head turned: 115 us (604 MB, 5.3 TB/s); 64 single tokens: 3.4 us.  With one piece in
// flight per lane, a division per piece and copying lanes behind rotating ones it was 75 and 157 us.
#include "common.h"

namespace {

enum { F32 = 0, BF16 = 1 };

struct Side { const void* in; void* out; int64_t ib, it, ih, ob, ot, oh; int heads; };
struct Args {
    Side q, k;
    const void* pos; const double* inv_freq;
    int64_t pb, pt, offset;
    int T, ntok, D, R, tb, pos64, copy, first;
    float magnitude, sign;
};

__device__ __forceinline__ float2 cos_sin(double pos, double f) {
    const double p = pos * f, lost = fma(pos, f, -p);
    const double n = rint(p * 0.63661977236758134308);                 // 2 / pi
    double rd = fma(-n, 1.57079632679489655800, p);                    // pi/2, first 53 bits
    rd = fma(-n, 6.12323399573676603587e-17, rd) + lost;               // ... and the next ones
    const int quarter = (int)(n - 4.0 * floor(n * 0.25));
    const float r = (float)rd, z = r * r;
    float s = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    s = fmaf(z, s, 8.33333333e-3f);
    s = fmaf(z, s, -0.166666667f);
    s = fmaf(r * z, s, r);
    float c = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
    c = fmaf(z, c, -1.38888889e-3f);
    c = fmaf(z, c, 4.16666667e-2f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    const float a = (quarter & 1) ? s : c, b = (quarter & 1) ? c : s;
    return make_float2((quarter == 1 || quarter == 2) ? -a : a, quarter >= 2 ? -b : b);
}

// V consecutive elements as fp32
template <int T, int V> struct Pack { float v[V]; };
template <int T, int V, bool NT> __device__ __forceinline__ Pack<T, V> load(const void* base, int64_t off) {
    Pack<T, V> r;
    if constexpr (T == F32) {
        const float* p = reinterpret_cast<const float*>(base) + off;
        if constexpr (V == 1) r.v[0] = p[0];
        else {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const float4 f = load_f4<NT>(p + i);
                r.v[i] = f.x; r.v[i + 1] = f.y; r.v[i + 2] = f.z; r.v[i + 3] = f.w;
            }
        }
    } else {
        const bf16_t* p = reinterpret_cast<const bf16_t*>(base) + off;
        if constexpr (V == 1) r.v[0] = bf2f(p[0]);
        else {
            const uint4 u = load_u4<NT>(p);
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { r.v[2 * i] = bf2f(w[i] & 0xffff); r.v[2 * i + 1] = bf2f(w[i] >> 16); }
        }
    }
    return r;
}
template <int T, int V> __device__ __forceinline__ void store(void* base, int64_t off, const Pack<T, V>& r) {
    if constexpr (T == F32) {
        float* p = reinterpret_cast<float*>(base) + off;
        if constexpr (V == 1) p[0] = r.v[0];
        else {
#pragma unroll
            for (int i = 0; i < V; i += 4) store_f4<false>(p + i, make_float4(r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]));
        }
    } else {
        bf16_t* p = reinterpret_cast<bf16_t*>(base) + off;
        if constexpr (V == 1) p[0] = f2bf(r.v[0]);
        else store_u4<false>(p, make_uint4(pack2bf(r.v[0], r.v[1]), pack2bf(r.v[2], r.v[3]), pack2bf(r.v[4], r.v[5]), pack2bf(r.v[6], r.v[7])));
    }
}

// V: elements per access (8 bf16 / 4 fp32, or 1 where an address, a stride or a width does not allow 16 bytes).
// threadIdx.x walks the pieces of one head -- first the rotated ones, then (copy) the ones that pass through -- and
// threadIdx.y the (token, head) pairs of the workgroup's tokens; blockIdx.y shares the heads of few tokens out.  A piece is one
// access, or two (TWO) where a pair's halves lie apart: at e and e2.  Two pieces are in flight per lane, their loads first:
// lanes that rotate and lanes that copy load and store together and part only for the arithmetic.
template <int T, bool HALF, int V, bool NT>
__global__ __launch_bounds__(256) void rotary_kernel(Args p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr bool TWO = HALF || V == 1;
    const int half = p.R >> 1, tok0 = p.first + blockIdx.x * p.tb, tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
    const int tokens = min(p.tb, p.ntok - tok0);
    int64_t* base = reinterpret_cast<int64_t*>(smem);                      // [tb][4]: where the token starts in q, qo, k, ko
    float2* table = reinterpret_cast<float2*>(smem + p.tb * 32);           // [tb][R/2]
    for (int i = tid; i < tokens * half; i += threads) {
        const int tl = i / half, f = i - tl * half, b = (tok0 + tl) / p.T, t = (tok0 + tl) - b * p.T;
        int64_t at = p.offset + t;
        if (p.pos) {
            const int64_t o = b * p.pb + t * p.pt;
            at = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[o] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[o];
        }
        const float2 cs = cos_sin((double)at, p.inv_freq[f]);
        table[i] = make_float2(cs.x * p.magnitude, cs.y * p.magnitude * p.sign);
        if (f == 0) {
            base[tl * 4 + 0] = b * p.q.ib + t * p.q.it;
            base[tl * 4 + 1] = b * p.q.ob + t * p.q.ot;
            base[tl * 4 + 2] = b * p.k.ib + t * p.k.it;
            base[tl * 4 + 3] = b * p.k.ob + t * p.k.ot;
        }
    }
    __syncthreads();
    const int heads = p.q.heads + p.k.heads, turned = TWO ? half / V : p.R / V;
    const int pieces = turned + (p.copy ? (TWO ? (p.D - p.R + 2 * V - 1) / (2 * V) : (p.D - p.R) / V) : 0);
    const int step = blockDim.y * gridDim.y, dt = step / heads, dh = step - dt * heads;
    for (int c = threadIdx.x; c < pieces; c += blockDim.x) {
        const bool turn = c < turned;
        int e = c * V, e2 = 0;
        if constexpr (HALF) {
            e = turn ? c * V : p.R + (c - turned) * 2 * V;
            e2 = turn ? half + c * V : e + V;
        } else if constexpr (TWO) {
            e = 2 * c;
            e2 = e + 1;
        }
        const bool second = TWO && e2 < p.D;
        int j = blockIdx.y * blockDim.y + threadIdx.y, tl = j / heads, h = j - tl * heads;
        while (tl < tokens) {
            int64_t at_out[2];
            void* out[2];
            const float2* cs[2];
            Pack<T, V> u[2], v[2];
            bool on[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                on[i] = tl < tokens;
                if (on[i]) {
                    const bool is_q = h < p.q.heads;
                    const int hh = is_q ? h : h - p.q.heads;
                    const void* in = is_q ? p.q.in : p.k.in;
                    const int64_t at = base[tl * 4 + (is_q ? 0 : 2)] + hh * (is_q ? p.q.ih : p.k.ih);
                    out[i] = is_q ? p.q.out : p.k.out;
                    at_out[i] = base[tl * 4 + (is_q ? 1 : 3)] + hh * (is_q ? p.q.oh : p.k.oh);
                    cs[i] = table + tl * half;
                    u[i] = load<T, V, NT>(in, at + e);
                    if (second) v[i] = load<T, V, NT>(in, at + e2);
                }
                tl += dt;
                h += dh;
                if (h >= heads) { h -= heads; ++tl; }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!on[i]) continue;
                if (turn) {
                    if constexpr (TWO) {
#pragma unroll
                        for (int x = 0; x < V; ++x) {
                            const float2 w = cs[i][c * V + x];
                            const float a = u[i].v[x], d = v[i].v[x];
                            u[i].v[x] = a * w.x - d * w.y;
                            v[i].v[x] = d * w.x + a * w.y;
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < V; x += 2) {
                            const float2 w = cs[i][(e + x) >> 1];
                            const float a = u[i].v[x], d = u[i].v[x + 1];
                            u[i].v[x] = a * w.x - d * w.y;
                            u[i].v[x + 1] = d * w.x + a * w.y;
                        }
                    }
                }
                store<T, V>(out[i], at_out[i] + e, u[i]);
                if (second) store<T, V>(out[i], at_out[i] + e2, v[i]);
            }
        }
    }
}

bool wide(const Side& s, int size) {
    const int64_t any = s.ib | s.it | s.ih | s.ob | s.ot | s.oh;
    return s.heads == 0 || (((uintptr_t)s.in | (uintptr_t)s.out) % 16 == 0 && any % (16 / size) == 0);
}

template <int T, bool HALF, int V> void launch(Args& a, hipStream_t st) {
    constexpr bool TWO = HALF || V == 1;
    const int half = a.R / 2, pieces = (TWO ? half : a.R) / V + (a.copy ? (TWO ? (a.D - a.R + 2 * V - 1) / (2 * V) : (a.D - a.R) / V) : 0);
    const int bx = pieces < 256 ? pieces : 256, by = 256 / bx, heads = a.q.heads + a.k.heads;
    // tokens per workgroup: enough that its 256 threads form one cosine and sine each, as long as that leaves 4 workgroups a CU
    a.tb = 256 / half < 1 ? 1 : 256 / half;
    while (a.tb > 1 && (a.ntok + a.tb - 1) / a.tb < 1024) a.tb >>= 1;
    const int blocks = (a.ntok + a.tb - 1) / a.tb, rounds = (a.tb * heads + by - 1) / by;
    int gy = 1;
    while (blocks * gy < 512 && gy * 2 <= rounds && gy < 64) gy *= 2;
    const size_t lds = (size_t)a.tb * (32 + half * sizeof(float2));
    // More than the Infinity Cache holds (256 MiB), and whole 128-byte lines an access: the inputs are read past the caches ("nt";
    // 32768 x 18 x 128 fp32 126 -> 115 us, interleaved bf16 58 -> 55).  Halves of 64 bytes share lines and lose: 63 -> 65.
    const size_t size = T == F32 ? 4 : 2;
    const bool nt = V > 1 && 2 * size * a.ntok * heads * a.D > ((size_t)256 << 20) && (!HALF || half * size % 128 == 0);
    // (a launch is at most 2^32 - 1 threads wide)
    const int most = 1 << 23;
    for (int b0 = 0; b0 < blocks; b0 += most) {
        const dim3 grid(blocks - b0 < most ? blocks - b0 : most, gy);
        a.first = b0 * a.tb;
        if (nt) hipLaunchKernelGGL((rotary_kernel<T, HALF, V, (V > 1)>), grid, dim3(bx, by), lds, st, a);
        else hipLaunchKernelGGL((rotary_kernel<T, HALF, V, false>), grid, dim3(bx, by), lds, st, a);
    }
}

}  // namespace

// strides: {in: batch, token, head; out: batch, token, head} of q, then of k, in elements
int getmi_rotary_impl(const void* q, void* qo, int hq, const void* k, void* ko, int hk, const int64_t* strides, int type, int B, int T, int D,
                      int R, const double* inv_freq, const void* pos, int pos64, int64_t pb, int64_t pt, int64_t offset, int interleaved,
                      int backward, float magnitude, hipStream_t st) {
    GETMI_CHECK_ARG(B >= 0 && T >= 0 && hq >= 0 && hk >= 0 && D > 0, "rotary: B=%d T=%d heads=%d,%d D=%d", B, T, hq, hk, D);
    GETMI_CHECK_ARG(R > 0 && R % 2 == 0 && R <= D && R <= 2048, "rotary: %d rotated columns of %d (even, at most 2048)", R, D);
    if (B == 0 || T == 0 || hq + hk == 0) return GETMI_OK;
    GETMI_CHECK_ARG((int64_t)B * T <= 0x7fff0000 && (int64_t)hq + hk <= 65536, "rotary: more than 0x7fff0000 tokens or 65536 heads");
    GETMI_CHECK_ARG(strides && inv_freq && (hq == 0 || (q && qo)) && (hk == 0 || (k && ko)), "rotary: null pointer");
    GETMI_CHECK_ARG(type == F32 || type == BF16, "rotary: types are 0 (fp32) and 1 (bf16)");
    Args a{};
    a.q = Side{q, qo, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], hq};
    a.k = Side{k, ko, strides[6], strides[7], strides[8], strides[9], strides[10], strides[11], hk};
    a.pos = pos; a.inv_freq = inv_freq; a.pb = pb; a.pt = pt; a.offset = offset;
    a.T = T; a.ntok = B * T; a.D = D; a.R = R; a.pos64 = pos64;
    // in place: the columns that pass through are there already
    a.copy = R < D && !((hq == 0 || q == qo) && (hk == 0 || k == ko));
    a.magnitude = magnitude; a.sign = backward ? -1.f : 1.f;
    const int size = type == F32 ? 4 : 2, v = 16 / size;
    // 16 bytes an access: every row, the second half of the rotated columns and the columns behind them start on 16 bytes
    const bool w = wide(a.q, size) && wide(a.k, size) && (interleaved ? R : R / 2) % v == 0 && (!a.copy || (D - R) % v == 0);
    if (type == F32) {
        if (interleaved) { if (w) launch<F32, false, 4>(a, st); else launch<F32, false, 1>(a, st); }
        else { if (w) launch<F32, true, 4>(a, st); else launch<F32, true, 1>(a, st); }
    } else {
        if (interleaved) { if (w) launch<BF16, false, 8>(a, st); else launch<BF16, false, 1>(a, st); }
        else { if (w) launch<BF16, true, 8>(a, st); else launch<BF16, true, 1>(a, st); }
    }
    GETMI_CHECK_LAUNCH("rotary");
    return GETMI_OK;
}
