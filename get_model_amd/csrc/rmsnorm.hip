// Root-mean-square norm with the residual's addition, its backward, and 8-bit (e4m3) outputs with one scale per 128 columns.
//
//   h = x + residual                y = w * h * rstd,  rstd = (mean(h^2) + eps)^(-1/2)
//   dh' = dh + rstd * (w*dy - hhat * mean(w*dy*hhat)),  hhat = h * rstd;   dw = sum over rows of dy * hhat
//   e4m3: per row and block of 128 columns  scale = 2^e, the smallest with max|y| <= 448 * 2^e,  q = e4m3(y / scale)
//
// One pass: a row lives in the registers of WPR waves (4 consecutive columns per lane and chunk: 16-byte loads of fp32, 8-byte
// loads of bf16), so every input is read once and every output written once.  HBM-bound.  All statistics, the sum h and the
// weight gradient are formed in fp32; y is formed from the unrounded fp32 h, and h is rounded once, to the residual's type.
// A power-of-two scale makes y / scale exact, so q carries the one rounding of the format itself, and it is what the
// matrix unit's own block scaling takes (gemm_fp8.hip).
//
// Measured, 51456 x 768, bf16 x on an fp32 residual, three operand sets in rotation (a 1-GiB copy reaches 5.0 TB/s): forward 72 us
// (12 bytes an element: 6.6 TB/s, part of it out of the Infinity Cache), 8-bit 71 us, backward 102 us (16 bytes, 6.2 TB/s) + 5 for
// the column sums' second stage.  Odd width, 51456 x 283 fp32: 20 / 35 us.  One row of 768: 2.1 us.  What got it there: the next
// row's loads in flight while a row is summed (94 -> 80), element-aligned wide accesses instead of single ones for odd widths (36 ->
// 20), nt loads for what the caches cannot hold, 1024 workgroups forward / 512 backward.
#include "fp8.h"

namespace {

enum { F32 = 0, BF16 = 1, NONE = 2, FP8 = 3 };

// ---- reductions on the DPP network: lanes 1, 2, 4 (half mirror) and 8 (mirror) apart inside a row of 16, then 16 and 32 ----
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ unsigned xor16(unsigned v) { return (unsigned)__builtin_amdgcn_ds_swizzle((int)v, 0x401f); }
__device__ __forceinline__ float row_sum64(float v) {
    v += __uint_as_float(dpp<0xb1>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x4e>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x140>(__float_as_uint(v)));
    v += __uint_as_float(xor16(__float_as_uint(v)));
    return v + __shfl_xor(v, 32, 64);
}
// maximum over the 32 lanes that hold one block of 128 columns.  On the bit patterns of |y|: NaN orders above infinity.
__device__ __forceinline__ unsigned max32(unsigned v) {
    v = max(v, dpp<0xb1>(v));
    v = max(v, dpp<0x4e>(v));
    v = max(v, dpp<0x141>(v));
    v = max(v, dpp<0x140>(v));
    return max(v, xor16(v));
}

template <int T> struct Elem { typedef float type; };
template <> struct Elem<BF16> { typedef bf16_t type; };

// Four consecutive columns of a row as they lie in memory.  Rows may start on any element (odd widths, views): the access is
// declared to be aligned to an element only, and the hardware takes a lane's 16 or 8 bytes from there in one instruction.
template <int T> struct Raw;
template <> struct Raw<F32> { typedef __attribute__((ext_vector_type(4), aligned(4))) float type; };
template <> struct Raw<BF16> { typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned short type; };

// n: how many of the four exist (<= 0: none, the result is zero)
template <int T, bool NT> __device__ __forceinline__ typename Raw<T>::type load_raw(const void* base, size_t off, int n) {
    typedef typename Raw<T>::type V;
    const typename Elem<T>::type* p = reinterpret_cast<const typename Elem<T>::type*>(base) + off;
    V v = {0, 0, 0, 0};
    if (n >= 4) {
        if constexpr (NT) v = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
        else v = *reinterpret_cast<const V*>(p);
    } else if (n > 0) {
        v[0] = p[0];
        if (n > 1) v[1] = p[1];
        if (n > 2) v[2] = p[2];
    }
    return v;
}
__device__ __forceinline__ float4 widen(Raw<F32>::type v) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float4 widen(Raw<BF16>::type v) { return make_float4(bf2f(v[0]), bf2f(v[1]), bf2f(v[2]), bf2f(v[3])); }
template <int T> __device__ __forceinline__ float4 load4(const void* base, size_t off, int n) { return widen(load_raw<T, false>(base, off, n)); }

template <int T> __device__ __forceinline__ void store4(void* base, size_t off, int n, float4 f) {
    typedef typename Raw<T>::type V;
    typename Elem<T>::type* p = reinterpret_cast<typename Elem<T>::type*>(base) + off;
    V v;
    if constexpr (T == F32) v = V{f.x, f.y, f.z, f.w};
    else {
        const uint2 u = pack4bf(f.x, f.y, f.z, f.w);
        v = V{(unsigned short)u.x, (unsigned short)(u.x >> 16), (unsigned short)u.y, (unsigned short)(u.y >> 16)};
    }
    if (n >= 4) {
        *reinterpret_cast<V*>(p) = v;
    } else if (n > 0) {
        p[0] = v[0];
        if (n > 1) p[1] = v[1];
        if (n > 2) p[2] = v[2];
    }
}

// sum over the WPR waves of a row; one LDS slot per wave, `red` is re-used every row (hence the second barrier)
__device__ __forceinline__ float join_waves(float v, float* red, int wave, int wpr) {
    if (wpr == 1) return v;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    const int first = wave - (wave & (wpr - 1));
    float s = 0.f;
    for (int i = 0; i < wpr; ++i) s += red[first + i];
    __syncthreads();
    return s;
}

struct FwdArgs {
    const void* x; const void* res; const float* w; void* y; void* h; float* rstd; unsigned char* scales;
    size_t ldx, ldr, ldq; int lds; int M, D, wpr; float eps; int norm;
};

// XT: type of x; RT: type of the residual and of h (NONE: there is none); YT: type of y (FP8: values and scales)
template <int XT, int RT, int YT, int NV, bool NT>
__global__ __launch_bounds__(1024) void rms_fwd_kernel(FwdArgs p) {
    __shared__ float red[16];
    constexpr int RTT = RT == NONE ? F32 : RT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nwaves = blockDim.x >> 6;
    const int rows = nwaves / p.wpr, part = wave & (p.wpr - 1), sub = wave / p.wpr, stride = gridDim.x * rows;
    int col[NV];
    float4 w[NV];
    typename Raw<XT>::type nx[NV];
    typename Raw<RTT>::type nr[NV];
    auto fetch = [&](int row) {      // the next row is on its way while this one is summed up
        if (row >= p.M) return;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            nx[v] = load_raw<XT, NT>(p.x, (size_t)row * p.ldx + col[v], p.D - col[v]);
            if constexpr (RT != NONE) nr[v] = load_raw<RTT, NT>(p.res, (size_t)row * p.ldr + col[v], p.D - col[v]);
        }
    };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        col[v] = ((v * p.wpr + part) * 64 + lane) * 4;
        nx[v] = typename Raw<XT>::type{0, 0, 0, 0};
        nr[v] = typename Raw<RTT>::type{0, 0, 0, 0};
        w[v] = p.norm ? load4<F32>(p.w, col[v], p.D - col[v]) : make_float4(1.f, 1.f, 1.f, 1.f);
    }
    fetch(blockIdx.x * rows + sub);
    // block-uniform trip count: rows past M take part in the barriers and touch no memory
    for (int base = blockIdx.x * rows; base < p.M; base += stride) {
        const int row = base + sub;
        const bool on = row < p.M;
        float4 a[NV];
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            a[v] = widen(nx[v]);
            if constexpr (RT != NONE) {
                const float4 r = widen(nr[v]);
                a[v].x += r.x; a[v].y += r.y; a[v].z += r.z; a[v].w += r.w;
            }
            s += a[v].x * a[v].x + a[v].y * a[v].y + a[v].z * a[v].z + a[v].w * a[v].w;
        }
        if (base + stride < p.M) fetch(row + stride);
        if constexpr (RT != NONE) {
#pragma unroll
            for (int v = 0; v < NV; ++v) store4<RTT>(p.h, (size_t)row * p.D + col[v], on ? p.D - col[v] : 0, a[v]);
        }
        float rs = 1.f;
        if (p.norm) {
            s = join_waves(row_sum64(s), red, wave, p.wpr);
            rs = 1.0f / sqrtf(s / (float)p.D + p.eps);
            if (p.rstd && on && part == 0 && lane == 0) p.rstd[row] = rs;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const float4 y = make_float4(a[v].x * rs * w[v].x, a[v].y * rs * w[v].y, a[v].z * rs * w[v].z, a[v].w * rs * w[v].w);
            if constexpr (YT == FP8) {
                const unsigned amax = max32(max(max(abs_bits(y.x), abs_bits(y.y)), max(abs_bits(y.z), abs_bits(y.w))));
                const unsigned byte = scale_byte(amax);
                if (on && col[v] < (int)p.ldq) {      // columns D .. ldq-1 are zeros: padding up to whole blocks
                    *reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(p.y) + (size_t)row * p.ldq + col[v]) =
                        pack4fp8(y.x, y.y, y.z, y.w, scale_value(byte), amax < 0x7f800000u);
                    if ((lane & 31) == 0) p.scales[(size_t)row * p.lds + (col[v] >> 7)] = (unsigned char)byte;
                }
            } else {
                store4<YT>(p.y, (size_t)row * p.D + col[v], on ? p.D - col[v] : 0, y);
            }
        }
    }
}

struct BwdArgs {
    const void* dy; const void* h; const float* rstd; const float* w; const void* dh; void* dx; void* dx2; float* partial;
    size_t ldh; int M, D, wpr;
};

// YT: type of dy; HT: type of h, dh and dx; dx2 (may be null): dx once more in bf16, for a bf16 x added to an fp32 residual
template <int YT, int HT, int NV, bool NT>
__global__ __launch_bounds__(1024) void rms_bwd_kernel(BwdArgs p) {
    extern __shared__ __attribute__((aligned(16))) float lds[];      // 16 join slots, then rows * D column sums where rows > 1
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nwaves = blockDim.x >> 6;
    const int rows = nwaves / p.wpr, part = wave & (p.wpr - 1), sub = wave / p.wpr, stride = gridDim.x * rows;
    int col[NV];
    float4 w[NV], aw[NV];
    typename Raw<YT>::type ny[NV];
    typename Raw<HT>::type nh[NV], nd[NV];
    float nrs = 0.f;
    auto fetch = [&](int row) {
        if (row >= p.M) return;
        nrs = p.rstd[row];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            ny[v] = load_raw<YT, NT>(p.dy, (size_t)row * p.D + col[v], p.D - col[v]);
            nh[v] = load_raw<HT, NT>(p.h, (size_t)row * p.ldh + col[v], p.D - col[v]);
            if (p.dh) nd[v] = load_raw<HT, NT>(p.dh, (size_t)row * p.D + col[v], p.D - col[v]);
        }
    };
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        col[v] = ((v * p.wpr + part) * 64 + lane) * 4;
        w[v] = load4<F32>(p.w, col[v], p.D - col[v]);
        aw[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        ny[v] = typename Raw<YT>::type{0, 0, 0, 0};
        nh[v] = nd[v] = typename Raw<HT>::type{0, 0, 0, 0};
    }
    fetch(blockIdx.x * rows + sub);
    for (int base = blockIdx.x * rows; base < p.M; base += stride) {
        const int row = base + sub;
        const bool on = row < p.M;
        const float rs = nrs;
        float4 g[NV], hh[NV], r[NV];
        float c = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            g[v] = on ? widen(ny[v]) : make_float4(0.f, 0.f, 0.f, 0.f);      // (a row past M adds nothing to the column sums)
            hh[v] = widen(nh[v]);
            r[v] = widen(nd[v]);
        }
        if (base + stride < p.M) fetch(row + stride);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            hh[v].x *= rs; hh[v].y *= rs; hh[v].z *= rs; hh[v].w *= rs;
            if (on) {
                aw[v].x += g[v].x * hh[v].x; aw[v].y += g[v].y * hh[v].y; aw[v].z += g[v].z * hh[v].z; aw[v].w += g[v].w * hh[v].w;
            }
            g[v].x *= w[v].x; g[v].y *= w[v].y; g[v].z *= w[v].z; g[v].w *= w[v].w;
            c += g[v].x * hh[v].x + g[v].y * hh[v].y + g[v].z * hh[v].z + g[v].w * hh[v].w;
        }
        c = join_waves(row_sum64(c), lds, wave, p.wpr) / (float)p.D;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int n = on ? p.D - col[v] : 0;
            const float4 d = make_float4(r[v].x + rs * (g[v].x - hh[v].x * c), r[v].y + rs * (g[v].y - hh[v].y * c),
                                         r[v].z + rs * (g[v].z - hh[v].z * c), r[v].w + rs * (g[v].w - hh[v].w * c));
            store4<HT>(p.dx, (size_t)row * p.D + col[v], n, d);
            if (p.dx2) store4<BF16>(p.dx2, (size_t)row * p.D + col[v], n, d);
        }
    }
    if (!p.partial) return;
    float* out = p.partial + (size_t)blockIdx.x * p.D;
    if (rows == 1) {      // every column belongs to one thread
#pragma unroll
        for (int v = 0; v < NV; ++v) store4<F32>(out, col[v], p.D - col[v], aw[v]);
        return;
    }
    float* sums = lds + 16;
#pragma unroll
    for (int v = 0; v < NV; ++v) store4<F32>(sums, (size_t)sub * p.D + col[v], p.D - col[v], aw[v]);
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += blockDim.x) {
        float t = 0.f;
        for (int k = 0; k < rows; ++k) t += sums[k * p.D + i];
        out[i] = t;
    }
}

// weight[N, K] -> e4m3 [N, ldq] and one scale per 128 x 128 block: one workgroup per block, 64 values a thread in registers
template <int WT>
__global__ __launch_bounds__(256) void quant_blocks_kernel(const void* w, size_t ldw, unsigned char* q, size_t ldq, unsigned char* scales,
                                                           int lds, int N, int K) {
    __shared__ unsigned red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 128 + (lane & 31) * 4, n = K - c;
    const int r0 = blockIdx.y * 128 + wave * 2 + (lane >> 5);
    typename Raw<WT>::type raw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) raw[i] = load_raw<WT, false>(w, (size_t)(r0 + 8 * i) * ldw + c, r0 + 8 * i < N ? n : 0);
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float4 v = widen(raw[i]);
        m = max(m, max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w))));
    }
    m = max32(m);
    m = max(m, (unsigned)__shfl_xor((int)m, 32, 64));
    if (lane == 0) red[wave] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    const unsigned byte = scale_byte(m);
    const float scale = scale_value(byte);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float4 v = widen(raw[i]);
        if (r0 + 8 * i < N)
            *reinterpret_cast<unsigned*>(q + (size_t)(r0 + 8 * i) * ldq + c) = pack4fp8(v.x, v.y, v.z, v.w, scale, m < 0x7f800000u);
    }
    if (threadIdx.x == 0) scales[(size_t)blockIdx.y * lds + blockIdx.x] = (unsigned char)byte;
}

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// waves per row and chunks per lane for `cols` columns
struct Shape { int wpr, nv, threads, rows; };
Shape shape_of(int cols, int M) {
    const int chunks = (cols + 255) / 256;
    Shape s;
    s.wpr = 1;
    while (s.wpr < 16 && (chunks + s.wpr - 1) / s.wpr > 3) s.wpr *= 2;      // (four chunks' backward spills: only past 12288 columns)
    if (M <= 512) while (s.wpr < chunks && s.wpr < 16) s.wpr *= 2;
    s.nv = (chunks + s.wpr - 1) / s.wpr;
    s.threads = s.wpr <= 4 ? 256 : s.wpr * 64;
    s.rows = s.threads / 64 / s.wpr;
    return s;
}
int grid_of(int M, int rows, int cap) {
    const int g = (int)(((int64_t)M + rows - 1) / rows);
    return g > cap ? cap : g;
}
int size_of(int type) { return type == F32 ? 4 : type == BF16 ? 2 : type == FP8 ? 1 : 0; }
// A call that moves well more than the Infinity Cache holds (256 MiB) reads its inputs past the caches ("nt"): 51456 x 768 in bf16 +
// fp32 forward 92 -> 72 us, 8-bit 86 -> 69, backward 121 -> 102.  A smaller one may find what the kernel before it wrote: there nt
// loads cost (51456 x 283 fp32 forward 20 -> 25 and backward 35 -> 42, 6000 x 6000 bf16 backward, 288 MB, 53 -> 59).  A template
// argument: a branch around the loads costs the small calls what nt loads cost them.
bool streams(size_t bytes) { return bytes > ((size_t)384 << 20); }
constexpr int MAX_D = 16384;      // 16 waves x 4 chunks x 256 columns
constexpr int MAX_M = 0x7fff0000;      // the row loops step past the end in 32 bits

template <int XT, int RT, int YT, bool NT> int launch_fwd(FwdArgs& a, const Shape& s, hipStream_t st) {
    const dim3 grid(grid_of(a.M, s.rows, 1024)), block(s.threads);
    switch (s.nv) {
        case 1: hipLaunchKernelGGL((rms_fwd_kernel<XT, RT, YT, 1, NT>), grid, block, 0, st, a); break;
        case 2: hipLaunchKernelGGL((rms_fwd_kernel<XT, RT, YT, 2, NT>), grid, block, 0, st, a); break;
        case 3: hipLaunchKernelGGL((rms_fwd_kernel<XT, RT, YT, 3, NT>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((rms_fwd_kernel<XT, RT, YT, 4, NT>), grid, block, 0, st, a); break;
    }
    GETMI_CHECK_LAUNCH("rmsnorm_fwd");
    return GETMI_OK;
}
template <int XT, int RT, int YT> int launch_fwd_nt(FwdArgs& a, const Shape& s, hipStream_t st) {
    return streams((size_t)a.M * a.D * (size_of(XT) + 2 * size_of(RT) + size_of(YT))) ? launch_fwd<XT, RT, YT, true>(a, s, st)
                                                                                       : launch_fwd<XT, RT, YT, false>(a, s, st);
}
template <int XT, int RT> int launch_fwd_y(FwdArgs& a, int yt, const Shape& s, hipStream_t st) {
    return yt == F32 ? launch_fwd_nt<XT, RT, F32>(a, s, st) : yt == BF16 ? launch_fwd_nt<XT, RT, BF16>(a, s, st)
                                                                       : launch_fwd_nt<XT, RT, FP8>(a, s, st);
}
int fwd(FwdArgs& a, int xt, int rt, int yt, hipStream_t st) {
    const Shape s = shape_of(yt == FP8 ? (int)a.ldq : a.D, a.M);
    a.wpr = s.wpr;
    if (xt == F32) return rt == NONE ? launch_fwd_y<F32, NONE>(a, yt, s, st) : launch_fwd_y<F32, F32>(a, yt, s, st);
    return rt == NONE ? launch_fwd_y<BF16, NONE>(a, yt, s, st)
         : rt == F32 ? launch_fwd_y<BF16, F32>(a, yt, s, st) : launch_fwd_y<BF16, BF16>(a, yt, s, st);
}

int bwd_grid(int M, const Shape& s) { return grid_of(M, s.rows, 512); }

}  // namespace

size_t getmi_rmsnorm_bwd_workspace_bytes_impl(int M, int D) {
    if (M <= 0 || D <= 0 || D > MAX_D) return 0;
    return (size_t)bwd_grid(M, shape_of(D, M)) * D * sizeof(float);
}

int getmi_rmsnorm_fwd_impl(const void* x, int xt, int64_t ldx, const void* res, int rt, int64_t ldr, const float* w, void* y, int yt,
                           void* h, float* rstd, int M, int D, float eps, hipStream_t st) {
    GETMI_CHECK_ARG(M >= 0 && M <= MAX_M && D > 0 && D <= MAX_D, "rmsnorm_fwd: M=%d D=%d (D <= %d)", M, D, MAX_D);
    if (M == 0) return GETMI_OK;
    GETMI_CHECK_ARG(x && w && y && (res == nullptr) == (h == nullptr), "rmsnorm_fwd: null pointer");
    GETMI_CHECK_ARG((xt == F32 || xt == BF16) && (yt == F32 || yt == BF16), "rmsnorm_fwd: types are 0 (fp32) and 1 (bf16)");
    GETMI_CHECK_ARG(!res || rt == F32 || (rt == BF16 && xt == BF16), "rmsnorm_fwd: the residual is fp32 or of x's type");
    GETMI_CHECK_ARG(ldx >= 0 && (!res || ldr >= 0) && eps >= 0.f, "rmsnorm_fwd: negative stride or eps");
    if (!res) rt = NONE;
    FwdArgs a{x, res, w, y, h, rstd, nullptr, (size_t)ldx, (size_t)ldr, 0, 0, M, D, 1, eps, 1};
    return fwd(a, xt, rt, yt, st);
}

int getmi_rmsnorm_fp8_impl(const void* x, int xt, int64_t ldx, const void* res, int rt, int64_t ldr, const float* w, void* q,
                           void* scales, int lds, void* h, int M, int D, float eps, hipStream_t st) {
    GETMI_CHECK_ARG(M >= 0 && M <= MAX_M && D > 0 && D <= MAX_D, "rmsnorm_fp8: M=%d D=%d (D <= %d)", M, D, MAX_D);
    if (M == 0) return GETMI_OK;
    GETMI_CHECK_ARG(x && q && scales && (res == nullptr) == (h == nullptr), "rmsnorm_fp8: null pointer");
    GETMI_CHECK_ARG(xt == F32 || xt == BF16, "rmsnorm_fp8: types are 0 (fp32) and 1 (bf16)");
    GETMI_CHECK_ARG(!res || rt == F32 || (rt == BF16 && xt == BF16), "rmsnorm_fp8: the residual is fp32 or of x's type");
    GETMI_CHECK_ARG(ldx >= 0 && (!res || ldr >= 0) && eps >= 0.f, "rmsnorm_fp8: negative stride or eps");
    GETMI_CHECK_ARG(w || !res, "rmsnorm_fp8: a residual without a norm");
    const int ldq = (D + 127) / 128 * 128;
    GETMI_CHECK_ARG(lds >= ldq / 128 && aligned(q, 4), "rmsnorm_fp8: scale row of %d bytes for %d blocks, or q not on 4 bytes", lds, ldq / 128);
    if (!res) rt = NONE;
    FwdArgs a{x, res, w, q, h, nullptr, reinterpret_cast<unsigned char*>(scales), (size_t)ldx, (size_t)ldr, (size_t)ldq, lds, M, D, 1, eps, w != nullptr};
    return fwd(a, xt, rt, FP8, st);
}

int getmi_quant_blocks_fp8_impl(const void* w, int wt, int64_t ldw, void* q, void* scales, int lds, int N, int K, hipStream_t st) {
    GETMI_CHECK_ARG(N >= 0 && N <= MAX_M && K > 0 && K <= MAX_M, "quant_blocks_fp8: N=%d K=%d", N, K);
    if (N == 0) return GETMI_OK;
    const int nb = (N + 127) / 128, kb = (K + 127) / 128;
    GETMI_CHECK_ARG(w && q && scales && (wt == F32 || wt == BF16) && ldw >= 0, "quant_blocks_fp8: null pointer, type or stride");
    GETMI_CHECK_ARG(lds >= kb && aligned(q, 4) && nb <= 65535, "quant_blocks_fp8: scale row of %d bytes for %d blocks, q not on 4 bytes or N too large", lds, kb);
    if (wt == F32) hipLaunchKernelGGL(quant_blocks_kernel<F32>, dim3(kb, nb), dim3(256), 0, st, w, (size_t)ldw, (unsigned char*)q, (size_t)kb * 128, (unsigned char*)scales, lds, N, K);
    else hipLaunchKernelGGL(quant_blocks_kernel<BF16>, dim3(kb, nb), dim3(256), 0, st, w, (size_t)ldw, (unsigned char*)q, (size_t)kb * 128, (unsigned char*)scales, lds, N, K);
    GETMI_CHECK_LAUNCH("quant_blocks_fp8");
    return GETMI_OK;
}

int getmi_colreduce_impl(const float* partial, float* out0, float* out1, float* out2, int R, int C, int accumulate, hipStream_t st);

template <int YT, int HT, bool NT> static void launch_bwd(const BwdArgs& a, const Shape& s, int grid, size_t lds, hipStream_t st) {
    switch (s.nv) {
        case 1: hipLaunchKernelGGL((rms_bwd_kernel<YT, HT, 1, NT>), dim3(grid), dim3(s.threads), lds, st, a); break;
        case 2: hipLaunchKernelGGL((rms_bwd_kernel<YT, HT, 2, NT>), dim3(grid), dim3(s.threads), lds, st, a); break;
        case 3: hipLaunchKernelGGL((rms_bwd_kernel<YT, HT, 3, NT>), dim3(grid), dim3(s.threads), lds, st, a); break;
        default: hipLaunchKernelGGL((rms_bwd_kernel<YT, HT, 4, NT>), dim3(grid), dim3(s.threads), lds, st, a); break;
    }
}
template <int YT, int HT> static void launch_bwd(const BwdArgs& a, const Shape& s, int grid, size_t lds, bool nt, hipStream_t st) {
    if (nt) launch_bwd<YT, HT, true>(a, s, grid, lds, st);
    else launch_bwd<YT, HT, false>(a, s, grid, lds, st);
}

int getmi_rmsnorm_bwd_impl(const void* dy, int yt, const void* h, int ht, int64_t ldh, const float* rstd, const float* w, const void* dh,
                           void* dx, void* dx2, float* dw, int M, int D, void* workspace, size_t workspace_bytes, hipStream_t st) {
    GETMI_CHECK_ARG(M > 0 && M <= MAX_M && D > 0 && D <= MAX_D, "rmsnorm_bwd: M=%d D=%d (D <= %d)", M, D, MAX_D);
    GETMI_CHECK_ARG(dy && h && rstd && w && dx && ldh >= 0, "rmsnorm_bwd: null pointer or negative stride");
    GETMI_CHECK_ARG((yt == F32 || yt == BF16) && (ht == F32 || ht == BF16), "rmsnorm_bwd: types are 0 (fp32) and 1 (bf16)");
    GETMI_CHECK_ARG(!dx2 || ht == F32, "rmsnorm_bwd: a second, bf16 dx only next to an fp32 one");
    GETMI_CHECK_ARG(!dw || (workspace && workspace_bytes >= getmi_rmsnorm_bwd_workspace_bytes_impl(M, D) && aligned(workspace, 16)),
                    "rmsnorm_bwd: dw needs a workspace of getmi_rmsnorm_bwd_workspace_bytes(M, D)");
    const Shape s = shape_of(D, M);
    const int g = bwd_grid(M, s);
    BwdArgs a{dy, h, rstd, w, dh, dx, dx2, dw ? reinterpret_cast<float*>(workspace) : nullptr, (size_t)ldh, M, D, s.wpr};
    const bool nt = streams((size_t)M * D * (size_of(yt) + (dh ? 3 : 2) * size_of(ht) + (dx2 ? 2 : 0)));
    const size_t lds = (16 + (s.rows > 1 ? (size_t)s.rows * D : 0)) * sizeof(float);      // at most 4 x 768 or 2 x 1536 columns
    if (yt == F32) { if (ht == F32) launch_bwd<F32, F32>(a, s, g, lds, nt, st); else launch_bwd<F32, BF16>(a, s, g, lds, nt, st); }
    else { if (ht == F32) launch_bwd<BF16, F32>(a, s, g, lds, nt, st); else launch_bwd<BF16, BF16>(a, s, g, lds, nt, st); }
    GETMI_CHECK_LAUNCH("rmsnorm_bwd");
    return dw ? getmi_colreduce_impl(a.partial, dw, nullptr, nullptr, g, D, 0, st) : GETMI_OK;
}
