// out[M,N] (bf16) = sum over blocks b of 128 columns:  2^sa[m,b] * 2^sb[n/128,b] * sum_{k in b} A[m,k] * B[n,k]   (+ bias[n])
// with e4m3 operands.  v_mfma_scale_f32_16x16x128_f8f6f4 takes one block of 128 in its depth and applies one power-of-two scale
// per row and 32 columns by itself, so the scales cost no vector instruction and the accumulators are plain fp32 sums.
#include "common.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;

struct Fp8Args {
    const unsigned char* A; const unsigned char* sa; const unsigned char* B; const unsigned char* sb; const float* bias; bf16_t* out;
    size_t lda, ldb, ldo; int lsa, lsb, M, N, K;
};

__device__ __forceinline__ i32x8 frag_global(const unsigned char* p) {
    typedef __attribute__((ext_vector_type(4))) int i32x4_t;
    const i32x4_t a = *reinterpret_cast<const i32x4_t*>(p), b = *reinterpret_cast<const i32x4_t*>(p + 16);
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ f32x4 mfma_fp8(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// One wave: 16 rows of A x 64 rows of B, operands straight from global memory.  The B rows are the matrix unit's rows and the A
// rows its columns, so a lane ends up with four consecutive n of one m.
__global__ __launch_bounds__(256) void gemm_fp8_kernel(Fp8Args p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, c = lane >> 4;
    const int m0 = blockIdx.y * 16, n0 = (blockIdx.x * 4 + wave) * 64;
    if (n0 >= p.N) return;
    const int m = min(m0 + r, p.M - 1);
    const unsigned char* a = p.A + (size_t)m * p.lda + c * 32;
    const unsigned char* sa = p.sa + (size_t)m * p.lsa;
    const unsigned char* sb = p.sb + (size_t)(n0 >> 7) * p.lsb;
    const unsigned char* b[4];
    f32x4 acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        b[t] = p.B + (size_t)min(n0 + t * 16 + r, p.N - 1) * p.ldb + c * 32;
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int k = 0; k < p.K; k += 128) {
        const i32x8 fa = frag_global(a + k);
        const int xa = sa[k >> 7], xb = sb[k >> 7];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = mfma_fp8(frag_global(b[t] + k), fa, acc[t], xb, xa);
    }
    if (m0 + r >= p.M) return;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + t * 16 + 4 * c + i;
            if (n < p.N) p.out[(size_t)(m0 + r) * p.ldo + n] = f2bf(acc[t][i] + (p.bias ? p.bias[n] : 0.f));
        }
}

int getmi_gemm_fp8_impl(const void* A, const void* sa, const void* B, const void* sb, const float* bias, void* out, int M, int N, int K,
                        int64_t lda, int64_t ldb, int64_t ldo, int lsa, int lsb, hipStream_t st) {
    GETMI_CHECK_ARG(M >= 0 && N >= 0 && K > 0 && K % 128 == 0, "gemm_fp8: M=%d N=%d K=%d (K is a multiple of 128: pad with zeros)", M, N, K);
    if (M == 0 || N == 0) return GETMI_OK;
    GETMI_CHECK_ARG(A && sa && B && sb && out, "gemm_fp8: null pointer");
    GETMI_CHECK_ARG(((uintptr_t)A | (uintptr_t)B | (uint64_t)lda | (uint64_t)ldb) % 16 == 0 && lda >= 0 && ldb >= 0 && ldo >= N,
                    "gemm_fp8: operand rows have to start on 16 bytes");
    GETMI_CHECK_ARG(((uintptr_t)sa | (uintptr_t)sb | (unsigned)lsa | (unsigned)lsb) % 4 == 0 && lsa >= 0 && lsb >= 0,
                    "gemm_fp8: scale rows have to start on 4 bytes");
    GETMI_CHECK_ARG((M + 15) / 16 <= 65535, "gemm_fp8: M=%d too large", M);
    Fp8Args p{(const unsigned char*)A, (const unsigned char*)sa, (const unsigned char*)B, (const unsigned char*)sb, bias, (bf16_t*)out,
              (size_t)lda, (size_t)ldb, (size_t)ldo, lsa, lsb, M, N, K};
    hipLaunchKernelGGL(gemm_fp8_kernel, dim3((N + 255) / 256, (M + 15) / 16), dim3(256), 0, st, p);
    GETMI_CHECK_LAUNCH("gemm_fp8");
    return GETMI_OK;
}
