// out[M,N] (bf16) = sum over blocks b of 128 columns:  2^sa[m,b] * 2^sb[n/128,b] * sum_{k in b} A[m,k] * B[n,k]   (+ bias[n])
// with e4m3 operands.  v_mfma_scale_f32_16x16x128_f8f6f4 takes one block of 128 in its depth and applies one power-of-two scale
// per row and 32 columns by itself, so the scales cost no vector instruction and the accumulators are plain fp32 sums.
#include "gemm_pipe.h"
#include <type_traits>

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

// ------------------------------------------------------------------------------------------------
// Large products: persistent 256 x 256 tiles, 8 waves (2 x 4, 128 x 64 each), one workgroup per CU.
//
// A K-tile is one scale block: 128 columns, 128 bytes a row -- byte for byte the image of a 64-deep bf16 K-tile, so it is staged
// and consumed like the bf16 kernel's (gemm.hip): four half-tiles (A0 B0 B1 A1) of 16 KiB by 16-byte LDS-DMA into an XOR-swizzled
// image, two K-tiles of ring, five half-tiles in flight across the barriers with counted vmcnt waits, four 64 x 32 quadrants per
// wave.  A quadrant is eight v_mfma_scale_f32_16x16x128 (a lane's 32 bytes are 16-byte chunks c and 4 + c of its row, for both
// operands alike, so the order inside the block does not matter).
// Scales: one 4-byte DMA per wave and K-tile beside the A0 half-tile brings the 4-byte word that holds the K-tile's scale byte, of
// 32 rows of A (lanes 0-31) and of the wave's own 128-column block of B (lanes 32-63).  The words are read at every fourth K-tile
// and shifted down a byte in between; the matrix unit takes the low byte.
// Stores are exactly E per wave and tile (inline asm, bounds-checked), so the next tile's counted waits leave them in flight.
// ------------------------------------------------------------------------------------------------
#define F8_SCALES 131072
#define F8_BIAS (F8_SCALES + 2 * 2048)
#define F8_STAGE (F8_BIAS + 2048)
#define F8_LDS (F8_STAGE + 8 * 2048)

__device__ __forceinline__ void glds4(const void* gsrc, void* lds_wave_base) {
    __builtin_amdgcn_global_load_lds(GLB_PTR(gsrc), LDS_PTR(lds_wave_base), 4, 0, 0);
}

template <int N> __device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N > 63 ? 63 : N) : "memory");
}
// at most `n` half-tiles (0..5) younger than the needed one, plus EXTRA stores, outstanding.  A0 half-tiles are 3 operations, the
// others 2; PH = 1, 2, 3: the phase, i.e. which kind follows the needed one (B1, A1, A0).
template <int PH, int EXTRA> __device__ __forceinline__ void wait_f8(int n) {
    constexpr int c[3][6] = {{0, 2, 4, 7, 9, 11}, {0, 2, 5, 7, 9, 11}, {0, 3, 5, 7, 9, 12}};
    if (n >= 5) wait_vm<c[PH - 1][5] + EXTRA>();
    else if (n == 4) wait_vm<c[PH - 1][4] + EXTRA>();
    else if (n == 3) wait_vm<c[PH - 1][3] + EXTRA>();
    else if (n == 2) wait_vm<c[PH - 1][2] + EXTRA>();
    else if (n == 1) wait_vm<c[PH - 1][1] + EXTRA>();
    else wait_vm<EXTRA>();
}

__device__ __forceinline__ i32x8 join8(u32x4 a, u32x4 b) {
    return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// RB: 16-row blocks of each wave's second 64-row half that are real output (4, 3, 2: tiles of 256, 224, 192 rows).
// ODD: rows of the output that do not start on 16 bytes, or N % 8 != 0: stored value by value.
template <int RB, bool ODD>
__global__ __launch_bounds__(512, 2) void gemm_fp8_256p_kernel(Fp8Args p, int ntiles, int group_n) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = 128 + 32 * RB, HW = BM / 2, E = (ODD ? 16 : 2) * (4 + RB);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int G = gridDim.x, nk = p.K >> 7;                     // nk >= 2 (host-checked)
    TileWalk walk;
    walk.init(xcd_remap(blockIdx.x, G), G, ntiles, (p.M + BM - 1) / BM, (p.N + 255) >> 8, group_n);
    const int ntl = walk.count, Gk = ntl * nk, Q = Gk << 2;
    const u32x4 rs = make_rsrc(p.out, (unsigned)(((size_t)(p.M - 1) * p.ldo + p.N) * 2));

    // byte offsets of the current and the next output tile: half-tile kinds 0 A0, 1 B0, 2 B1, 3 A1; [4]: the scale words
    unsigned cur[4][2], nxt[4][2], curs, nxts;
    int dst[4][2];
    const unsigned char* sbase = lane < 32 ? p.sa : p.sb;
    auto tile_offsets = [&](int it, unsigned (&o)[4][2], unsigned& os) {
        int tm, tn;
        walk.decode(it, tm, tn);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const int hr = (wave * 2 + jj) * 8 + (lane >> 3);
                if (j == 0 || j == 3) {
                    const int row = ((hr >> 6) << 7) + (j == 3) * 64 + (hr & 63);
                    const int g = min(tm * BM + ((hr >> 6) ? HW : 0) + (j == 3) * 64 + (hr & 63), p.M - 1);
                    o[j][jj] = (unsigned)((size_t)g * p.lda) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
                } else {
                    const int row = ((hr >> 5) << 6) + (j - 1) * 32 + (hr & 31);
                    const int g = min((tn << 8) + row, p.N - 1);
                    o[j][jj] = (unsigned)((size_t)g * p.ldb) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
                }
            }
        const int R = wave * 32 + (lane & 31);
        os = lane < 32 ? (unsigned)min(tm * BM + ((R >> 7) ? HW : 0) + (R & 127), p.M - 1) * (unsigned)p.lsa
                       : (unsigned)min(tn * 2 + (wn >> 1), (p.N - 1) >> 7) * (unsigned)p.lsb;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
            const int hr0 = (wave * 2 + jj) * 8;
            if (j == 0 || j == 3) dst[j][jj] = (((hr0 >> 6) << 7) + (j == 3) * 64 + (hr0 & 63)) * 128;
            else dst[j][jj] = 32768 + (((hr0 >> 5) << 6) + (j - 1) * 32 + (hr0 & 31)) * 128;
        }
    tile_offsets(0, cur, curs);
    tile_offsets(1, nxt, nxts);
    int tile_g0 = 0, it = 0;
    const char* baseA = reinterpret_cast<const char*>(p.A);
    const char* baseB = reinterpret_cast<const char*>(p.B);
#define F8_ISSUE_(gi_, koff_, O, OS, J)                                                                    \
    do {                                                                                                   \
        char* b_ = smem + ((gi_ & 1) << 16);                                                               \
        const char* base_ = ((J) == 0 || (J) == 3) ? baseA : baseB;                                        \
        glds16(base_ + (size_t)((O(J, 0)) + koff_), b_ + dst[J][0]);                                       \
        glds16(base_ + (size_t)((O(J, 1)) + koff_), b_ + dst[J][1]);                                       \
        if ((J) == 0) glds4(sbase + (size_t)(OS + ((koff_ >> 9) << 2)), smem + F8_SCALES + ((gi_ & 1) << 11) + wave * 256); \
    } while (0)
    // half-tile J of K-tile gi of the workgroup's stream, which lies in the current or the next output tile
#define F8_ISSUE(gi, J)                                                                                    \
    do {                                                                                                   \
        const int gi_ = (gi);                                                                              \
        const bool nx_ = gi_ >= tile_g0 + nk;                                                              \
        const unsigned koff_ = (unsigned)(gi_ - tile_g0 - (nx_ ? nk : 0)) * 128u;                          \
        F8_ISSUE_(gi_, koff_, F8_SEL, (nx_ ? nxts : curs), J);                                             \
    } while (0)
#define F8_SEL(J, i) (nx_ ? nxt[J][i] : cur[J][i])
#define F8_CUR(J, i) cur[J][i]
    // ... which is known to lie in the current one
#define F8_ISSUE_CUR(gi, J)                                                                                \
    do {                                                                                                   \
        const int gi_ = (gi);                                                                              \
        const unsigned koff_ = (unsigned)(gi_ - tile_g0) * 128u;                                           \
        F8_ISSUE_(gi_, koff_, F8_CUR, curs, J);                                                            \
    } while (0)

    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int r = lane & 15, c = lane >> 4, fsw = (r >> 1) & 7;
    const unsigned lds0 = lds_addr(smem);
    unsigned la[2], lb[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const int off = r * 128 + (((4 * ks + c) ^ fsw) << 4);
        la[ks] = lds0 + wm * 16384 + off;
        lb[ks] = lds0 + 32768 + wn * 8192 + off;
    }
    const unsigned lsa = lds0 + F8_SCALES + wm * 1024 + r * 4, lsb = lds0 + F8_SCALES + wave * 256 + 128;
    char* bias_img = smem + F8_BIAS + wave * 256;      // this wave's 64 columns
    const unsigned stage = lds0 + F8_STAGE + wave * 2048;
    auto stage_bias = [&](int iter) {
        int tm, tn;
        walk.decode(iter, tm, tn);
        glds4(p.bias + min((tn << 8) + wn * 64 + lane, p.N - 1), bias_img);
    };
    if (p.bias) stage_bias(0);
    F8_ISSUE(0, 0); F8_ISSUE(0, 1); F8_ISSUE(0, 2); F8_ISSUE(0, 3);
    F8_ISSUE(1, 0); F8_ISSUE(1, 1); F8_ISSUE(1, 2);

    u32x4 fa[4][2], fb0[2][2], fb1[2][2];
    unsigned sa[8], sb = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sa[i] = 0;
    // fragment reads in inline asm with counted lgkmcnt waits: their destinations are undefined until the wait that names them
#define F8_RD(dst, addr, OFF) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(dst) : "v"(addr), "n"(OFF) : "memory")
#define F8_RD4(dst, addr, OFF) asm volatile("ds_read_b32 %0, %1 offset:%2" : "=&v"(dst) : "v"(addr), "n"(OFF) : "memory")
#define F8_LG2(N, x) asm volatile("s_waitcnt lgkmcnt(" #N ")" : "+v"(x[0]), "+v"(x[1]) : : "memory")
#define F8_LG4(N, x, y) asm volatile("s_waitcnt lgkmcnt(" #N ")" : "+v"(x[0]), "+v"(x[1]), "+v"(y[0]), "+v"(y[1]) : : "memory")
#define F8_RD_A(MH, mt) F8_RD(fa[mt][0], a0, (MH)*8192 + (mt)*2048); F8_RD(fa[mt][1], a1, (MH)*8192 + (mt)*2048);
#define F8_RD_B(FB, NH, nt) F8_RD(FB[nt][0], b0, (NH)*4096 + (nt)*2048); F8_RD(FB[nt][1], b1, (NH)*4096 + (nt)*2048);
#define F8_MM1(MH, NH, FB, mt, nt)                                                                         \
    if constexpr ((MH) == 0 || (mt) < RB) {                                                                \
        acc[(MH)*4 + mt][(NH)*2 + nt] = mfma_fp8(join8(FB[nt][0], FB[nt][1]), join8(fa[mt][0], fa[mt][1]), \
                                                 acc[(MH)*4 + mt][(NH)*2 + nt], (int)sb, (int)sa[(MH)*4 + mt]); \
        asm volatile("" : "+v"(acc[(MH)*4 + mt][(NH)*2 + nt]));      /* keeps it in its phase */           \
    }
#define F8_MM(MH, NH, FB, mt)                                                                              \
    F8_MM1(MH, NH, FB, mt, 0) F8_MM1(MH, NH, FB, mt, 1) __builtin_amdgcn_sched_barrier(0);
    int win = 0;      // > 0 while the needed half-tile predates the last epilogue's stores
    // the wait of phase PH: five half-tiles (plus the last epilogue's stores in the phases that still precede them) stay in flight,
    // fewer where the stream ends
#define F8_WAIT(PH, last)                                                                                  \
    do {                                                                                                   \
        if constexpr (MODE == HEAD || (MODE == SECOND && (PH) < 3)) wait_f8<PH, E>(5);                     \
        else if constexpr (MODE != END) wait_f8<PH, 0>(5);                                                 \
        else if (win > 0) { wait_f8<PH, E>(min(phi + (last), Q - 1) - (phi + (PH))); --win; }              \
        else wait_f8<PH, 0>(min(phi + (last), Q - 1) - (phi + (PH)));                                      \
    } while (0)
#define F8_NEXT(d, J)                                                                                      \
    do {                                                                                                   \
        if constexpr (MODE == MID) F8_ISSUE_CUR(g + (d), J);                                               \
        else if constexpr (MODE != END) F8_ISSUE(g + (d), J);                                              \
        else if (g + (d) < Gk) F8_ISSUE(g + (d), J);                                                       \
    } while (0)
    // One K-tile.  MID: everything it issues lies in the same output tile.  HEAD, SECOND: the first two after an epilogue.
    // LAST: what it issues may lie in the next output tile.  END: the stream ends within two K-tiles.
    enum { MID, HEAD, SECOND, LAST, END };
    auto ktile = [&](int g, auto mode_) {
        constexpr int MODE = decltype(mode_)::value;
        const unsigned bo = (unsigned)(g & 1) << 16, so = (unsigned)(g & 1) << 11;
        const unsigned a0 = la[0] + bo, a1 = la[1] + bo, b0 = lb[0] + bo, b1 = lb[1] + bo;
        const int phi = g << 2;
        // ---- P1: A-half0 x B-half0 ----
        F8_WAIT(1, 6);
        phase_barrier();
        F8_NEXT(1, 3);
        if (((g - tile_g0) & 3) == 0) {
            const unsigned x = lsa + so, y = lsb + so;
            F8_RD4(sb, y, 0);
            F8_RD4(sa[0], x, 0); F8_RD4(sa[1], x, 64); F8_RD4(sa[2], x, 256); F8_RD4(sa[3], x, 320);
            F8_RD4(sa[4], x, 512); F8_RD4(sa[5], x, 576); F8_RD4(sa[6], x, 768); F8_RD4(sa[7], x, 832);
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(sb), "+v"(sa[0]), "+v"(sa[1]), "+v"(sa[2]), "+v"(sa[3]), "+v"(sa[4]), "+v"(sa[5]),
                         "+v"(sa[6]), "+v"(sa[7]) : : "memory");
        } else {
            sb >>= 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) sa[i] >>= 8;
        }
        F8_RD_B(fb0, 0, 0) F8_RD_A(0, 0) F8_RD_B(fb0, 0, 1) F8_RD_A(0, 1) F8_RD_A(0, 2) F8_RD_A(0, 3)
        F8_LG4(8, fb0[0], fa[0]); F8_MM1(0, 0, fb0, 0, 0) __builtin_amdgcn_sched_barrier(0);
        F8_LG2(6, fb0[1]); F8_MM1(0, 0, fb0, 0, 1) __builtin_amdgcn_sched_barrier(0);
        F8_LG2(4, fa[1]); F8_MM(0, 0, fb0, 1)
        F8_LG2(2, fa[2]); F8_MM(0, 0, fb0, 2)
        F8_LG2(0, fa[3]); F8_MM(0, 0, fb0, 3)
        // ---- P2: A-half0 (in registers) x B-half1 ----
        F8_WAIT(2, 7);
        phase_barrier();
        F8_NEXT(2, 0);
        F8_RD_B(fb1, 1, 0) F8_RD_B(fb1, 1, 1)
        F8_LG2(2, fb1[0]); F8_MM1(0, 1, fb1, 0, 0) F8_MM1(0, 1, fb1, 1, 0) F8_MM1(0, 1, fb1, 2, 0) F8_MM1(0, 1, fb1, 3, 0)
        __builtin_amdgcn_sched_barrier(0);
        F8_LG2(0, fb1[1]); F8_MM1(0, 1, fb1, 0, 1) F8_MM1(0, 1, fb1, 1, 1) F8_MM1(0, 1, fb1, 2, 1) F8_MM1(0, 1, fb1, 3, 1)
        __builtin_amdgcn_sched_barrier(0);
        // ---- P3: A-half1 x B-half1 (in registers) ----
        F8_WAIT(3, 8);
        phase_barrier();
        F8_NEXT(2, 1);
        F8_RD_A(1, 0) F8_RD_A(1, 1) F8_RD_A(1, 2) F8_RD_A(1, 3)
        F8_LG2(6, fa[0]); F8_MM(1, 1, fb1, 0)
        F8_LG2(4, fa[1]); F8_MM(1, 1, fb1, 1)
        F8_LG2(2, fa[2]); F8_MM(1, 1, fb1, 2)
        F8_LG2(0, fa[3]); F8_MM(1, 1, fb1, 3)
        // ---- P4: A-half1 x B-half0, both in registers (no barrier) ----
        F8_NEXT(2, 2);
        F8_MM(1, 0, fb0, 0) F8_MM(1, 0, fb0, 1) F8_MM(1, 0, fb0, 2) F8_MM(1, 0, fb0, 3)
        if constexpr (MODE == HEAD) win = 2;
        if constexpr (MODE == SECOND) win = 0;
    };

    for (int t = 0; t < ntl; ++t) {
        int k = 0;
        const int kend = t + 1 < ntl ? nk : nk - 2;      // K-tiles whose issues all lie inside the stream
        if (t > 0) {
            if (k < kend) { ktile(tile_g0 + k, std::integral_constant<int, HEAD>{}); ++k; }
            if (k < kend) { ktile(tile_g0 + k, std::integral_constant<int, SECOND>{}); ++k; }
        }
        for (; k + 2 < nk; ++k) ktile(tile_g0 + k, std::integral_constant<int, MID>{});
        for (; k < kend; ++k) ktile(tile_g0 + k, std::integral_constant<int, LAST>{});
        for (; k < nk; ++k) ktile(tile_g0 + k, std::integral_constant<int, END>{});
        // (the lane's number once more, opaque: what is derived from it here shall not occupy registers in the main loop)
        int el = threadIdx.x & 63;
        asm volatile("" : "+v"(el));
        const int er = el & 15, ec = el >> 4, rrow = el >> 3, rch = el & 7;
        const unsigned wa = stage + er * 128 + ((((unsigned)(ec >> 1) ^ (er & 7)) << 4) | ((ec & 1) << 3));
        const unsigned ra = stage + rrow * 128 + ((rch ^ (rrow & 7)) << 4);
        int tm, tn;
        walk.decode(it, tm, tn);
        const int m0w = tm * BM + wm * HW, n0w = (tn << 8) + wn * 64, mend = min(p.M, m0w + HW);
        f32x4 bv[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) bv[b] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (p.bias)      // complete: older than the half-tiles that the last counted waits waited for
            asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:64\n\tds_read_b128 %2, %4 offset:128\n\t"
                         "ds_read_b128 %3, %4 offset:192\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(bv[0]), "=&v"(bv[1]), "=&v"(bv[2]), "=&v"(bv[3])
                         : "v"(lds_addr(bias_img) + ec * 16) : "memory");
#pragma unroll
        for (int a = 0; a < 4 + RB; ++a) {
            u32x2 q[4];
            u32x4 d[2];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const f32x4 v = acc[a][b] + bv[b];
                q[b] = (u32x2){pack2bf(v[0], v[1]), pack2bf(v[2], v[3])};
            }
            stage_w64x4_r128x2(wa, ra, q[0], q[1], q[2], q[3], d[0], d[1]);
#pragma unroll
            for (int ps = 0; ps < 2; ++ps) {
                const int m = m0w + a * 16 + ps * 8 + rrow, n = n0w + rch * 8;
                const unsigned off = (unsigned)(((size_t)m * p.ldo + n) * 2);
                if constexpr (!ODD) st_b128<true>(d[ps], (m < mend && n < p.N) ? off : OOB_OFF, rs);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const unsigned o = (m < mend && n + j < p.N) ? off + 2 * j : OOB_OFF;
                        const unsigned v = d[ps][j >> 1];
                        if (j & 1) asm volatile("buffer_store_short_d16_hi %0, %1, %2, 0 offen\n\ts_nop 1" ::"v"(v), "v"(o), "s"(rs) : "memory");
                        else asm volatile("buffer_store_short %0, %1, %2, 0 offen\n\ts_nop 1" ::"v"(v), "v"(o), "s"(rs) : "memory");
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        ++it;
        tile_g0 += nk;
#pragma unroll
        for (int j = 0; j < 4; ++j) { cur[j][0] = nxt[j][0]; cur[j][1] = nxt[j][1]; }
        curs = nxts;
        tile_offsets(it + 1, nxt, nxts);
        if (p.bias && it < ntl) stage_bias(it);
        win = 5;
    }
#undef F8_ISSUE
#undef F8_ISSUE_
#undef F8_ISSUE_CUR
#undef F8_SEL
#undef F8_CUR
#undef F8_RD
#undef F8_RD4
#undef F8_LG2
#undef F8_LG4
#undef F8_RD_A
#undef F8_RD_B
#undef F8_MM1
#undef F8_MM
#undef F8_WAIT
#undef F8_NEXT
}

int getmi_cu_budget();

// Columns of output tiles whose B blocks an XCD keeps in its L2 from round to round (see TileWalk): as many as fit into 2.5 MB,
// weighed against reading A once per group.
static int pick_group(int M, int N, int K, int tile_m, int grid) {
    const int tiles_n = (N + 255) / 256, tiles_m = (M + tile_m - 1) / tile_m;
    if (grid % 8 != 0) return 0;
    const double a_bytes = (double)M * K, blk = 256.0 * K, rounds = (double)tiles_m * tiles_n / grid;
    double best = 0;
    int best_g = tiles_n;
    for (int g = 1; g <= tiles_n; ++g) {
        const double cost = a_bytes * ((tiles_n + g - 1) / g) + (g * blk <= 2.5e6 ? 8.0 : 8.0 * (rounds < 1 ? 1 : rounds)) * g * blk;
        if (best == 0 || cost < best - 1.0) { best = cost; best_g = g; }
    }
    return best_g;
}

template <int RB, bool ODD> static int launch_256p(const Fp8Args& p, hipStream_t st) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_fp8_256p_kernel<RB, ODD>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, F8_LDS);
    (void)attr;
    constexpr int BM = 128 + 32 * RB;
    const int ntiles = ((p.M + BM - 1) / BM) * ((p.N + 255) / 256), cus = getmi_cu_budget(), grid = ntiles < cus ? ntiles : cus;
    hipLaunchKernelGGL((gemm_fp8_256p_kernel<RB, ODD>), dim3(grid), dim3(512), F8_LDS, st, p, ntiles, pick_group(p.M, p.N, p.K, BM, grid));
    GETMI_CHECK_LAUNCH("gemm_fp8");
    return GETMI_OK;
}
template <bool ODD> static int launch_big(const Fp8Args& p, hipStream_t st) {
    // tile height: rounds of the CUs x the time of a round (256 rows: 1, 224: 0.93, 192: 0.87 -- the bf16 kernel's measure)
    const int cus = getmi_cu_budget(), tn = (p.N + 255) / 256;
    const double t[3] = {0.87, 0.93, 1.0};
    int best = 4;
    double cost = 0;
    for (int rb = 4; rb >= 2; --rb) {
        const int bm = 128 + 32 * rb, tiles = ((p.M + bm - 1) / bm) * tn;
        const double c = (double)((tiles + cus - 1) / cus) * t[rb - 2];
        if (cost == 0 || c < cost - 1e-9) { cost = c; best = rb; }
    }
    return best == 4 ? launch_256p<4, ODD>(p, st) : best == 3 ? launch_256p<3, ODD>(p, st) : launch_256p<2, ODD>(p, st);
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
    const size_t lim = 0xF0000000ull;      // the large kernel addresses each operand with 32 bits
    const bool fits = (size_t)M * lda < lim && (size_t)N * ldb < lim && (size_t)M * ldo * 2 < lim && (size_t)M * lsa < lim && (size_t)N * lsb < lim;
    if (K >= 256 && M >= 128 && (int64_t)((M + 255) / 256) * ((N + 255) / 256) >= 64 && fits)
        return (ldo % 8 == 0 && N % 8 == 0 && (uintptr_t)out % 16 == 0) ? launch_big<false>(p, st) : launch_big<true>(p, st);
    hipLaunchKernelGGL(gemm_fp8_kernel, dim3((N + 255) / 256, (M + 15) / 16), dim3(256), 0, st, p);
    GETMI_CHECK_LAUNCH("gemm_fp8");
    return GETMI_OK;
}
