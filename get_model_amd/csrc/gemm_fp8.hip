// out[M,N] (bf16) = sum over blocks b of 128 columns:  2^sa[m,b] * 2^sb[n/128,b] * sum_{k in b} A[m,k] * B[n,k]   (+ bias[n])
// with e4m3 operands.  v_mfma_scale_f32_16x16x128_f8f6f4 takes one block of 128 in its depth and applies one power-of-two scale
// per row and 32 columns by itself, so the scales cost no vector instruction and the accumulators are plain fp32 sums.
#include "fp8.h"
#include "gemm_pipe.h"
#include <algorithm>
#include <atomic>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) int i32x8;

struct Fp8Args {
    const unsigned char* A; const unsigned char* sa; const unsigned char* B; const unsigned char* sb; const float* bias; bf16_t* out;
    size_t lda, ldb, ldo; int lsa, lsb, M, N, K, Ka;
};

__device__ __forceinline__ f32x4 mfma_fp8(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
__device__ __forceinline__ i32x8 join8(u32x4 a, u32x4 b) {
    return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}
// A lane's 32 bytes of one block of its row: 16-byte chunks c and 4 + c (each load of a wave then covers 64 consecutive bytes of
// 16 rows).  Both operands are read alike, so the order inside the block does not matter.
__device__ __forceinline__ i32x8 frag_global(const unsigned char* p) {
    return join8(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 64));
}
// four consecutive outputs of row m from column n on; gran: how many columns of a row can be stored at once (see granularity())
__device__ __forceinline__ void store_out4(const Fp8Args& p, int m, int n, f32x4 v, int gran) {
    if (m >= p.M || n >= p.N) return;
    bf16_t* o = p.out + (size_t)m * p.ldo + n;
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += p.bias[min(n + i, p.N - 1)];
    }
    if (gran >= 4) {
        *reinterpret_cast<uint2*>(o) = pack4bf(v[0], v[1], v[2], v[3]);
    } else if (gran == 2) {
        *reinterpret_cast<unsigned*>(o) = pack2bf(v[0], v[1]);
        if (n + 2 < p.N) *reinterpret_cast<unsigned*>(o + 2) = pack2bf(v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) o[i] = f2bf(v[i]);
    }
}

// ------------------------------------------------------------------------------------------------
// Few rows (M <= 16 MT): the weights' bytes are the time.  A workgroup owns 16 NT rows of B over the whole depth; its W waves take
// every W-th block of 128 each, straight from global memory into the matrix unit (nothing is reused, so LDS would only delay it),
// and the W partial sums are joined in LDS in a fixed order.  The B rows are the matrix unit's rows and the A rows its columns, so
// a lane ends up with four consecutive n of one m.
// ------------------------------------------------------------------------------------------------
enum { A_F32 = 0, A_BF16 = 1, A_FP8 = 2 };

// Eight consecutive columns of a 16- or 32-bit row as they lie in memory, of which n exist (the others are zero).  Rows may start on
// any element.  grow(): the running maximum of the magnitudes; amax(): its fp32 bit pattern; pack(h): half h as e4m3.
template <int AT> struct Eight;
template <> struct Eight<A_BF16> {
    typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned V;
    V v;
    __device__ __forceinline__ void load(const unsigned char* row, int col, int n) {
        const bf16_t* p = reinterpret_cast<const bf16_t*>(row) + col;
        v = V{0, 0, 0, 0};
        if (n >= 8) v = *reinterpret_cast<const V*>(p);
        else if (n > 0)      // (all loads, then the choice: a load under a condition of its own would wait for the one before)
#pragma unroll
            for (int i = 0; i < 7; ++i) { const unsigned e = p[min(i, n - 1)]; v[i >> 1] |= i < n ? e << (i & 1) * 16 : 0; }
    }
    __device__ __forceinline__ unsigned grow(unsigned m) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max_abs_bf16(m, v[i]);
        return m;
    }
    static __device__ __forceinline__ unsigned amax(unsigned m) { return abs_bits_bf16(m); }
    __device__ __forceinline__ unsigned pack(int h, unsigned byte, bool finite) const {
        return pack4fp8_bf16(v[2 * h], v[2 * h + 1], scale_value(byte), finite);
    }
};
template <> struct Eight<A_F32> {
    typedef __attribute__((ext_vector_type(4), aligned(4))) float V;
    V v[2];
    __device__ __forceinline__ void load(const unsigned char* row, int col, int n) {
        const float* p = reinterpret_cast<const float*>(row) + col;
        v[0] = v[1] = V{0.f, 0.f, 0.f, 0.f};
        if (n >= 8) { v[0] = *reinterpret_cast<const V*>(p); v[1] = *reinterpret_cast<const V*>(p + 4); }
        else if (n > 0)
#pragma unroll
            for (int i = 0; i < 7; ++i) { const float e = p[min(i, n - 1)]; v[i >> 2][i & 3] = i < n ? e : 0.f; }
    }
    __device__ __forceinline__ unsigned grow(unsigned m) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i >> 2][i & 3]));
        return m;
    }
    static __device__ __forceinline__ unsigned amax(unsigned m) { return m; }
    __device__ __forceinline__ unsigned pack(int h, unsigned byte, bool finite) const {
        return pack4fp8(v[h][0], v[h][1], v[h][2], v[h][3], scale_value(byte), finite);
    }
};
template <> struct Eight<A_FP8> {};

// A lane's 32 values of one block of its row, quantised on the way: the block's maximum is the maximum over the four lanes that hold
// it (16 and 32 apart).  The same values and scale as the row quantiser's.
template <int AT> __device__ __forceinline__ i32x8 frag_quantised(const unsigned char* row, int kb, int c, int K, unsigned& scale) {
    const int col = kb * 128 + c * 16;
    Eight<AT> e[4];
    unsigned m = 0;
    if (kb * 128 + 128 <= K) {      // (the same for all: no branch per piece but in the last block)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i].load(row, col + (i >> 1) * 64 + (i & 1) * 8, 8);
    } else
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i].load(row, col + (i >> 1) * 64 + (i & 1) * 8, K - col - (i >> 1) * 64 - (i & 1) * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = e[i].grow(m);
    m = Eight<AT>::amax(m);
    m = max(m, (unsigned)__builtin_amdgcn_ds_swizzle((int)m, 0x401f));
    m = max(m, (unsigned)__shfl_xor((int)m, 32, 64));
    scale = scale_byte(m);
    const bool finite = m < 0x7f800000u;
    i32x8 f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (int)e[i >> 1].pack(i & 1, scale, finite);
    return f;
}

// AT: e4m3 rows with scales, or 16- / 32-bit rows (p.sa unused, p.lda in bytes, p.Ka columns) that every workgroup quantises for
// itself: one launch for a token's linear.
template <int MT, int NT, int AT>
__global__ __launch_bounds__(1024) void gemm_fp8_rows_kernel(Fp8Args p, int gran) {
    extern __shared__ __attribute__((aligned(16))) f32x4 part[];      // [W][NT * MT][64]
    const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6, nkb = p.K >> 7;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const unsigned char *a[MT], *b[NT], *sa[MT];
    const unsigned char* sb = p.sb + (size_t)(n0 >> 7) * p.lsb;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const size_t m = min(m0 + j * 16 + r, p.M - 1);
        a[j] = p.A + m * p.lda + (AT == A_FP8 ? c * 16 : 0);
        sa[j] = p.sa + (AT == A_FP8 ? m * p.lsa : 0);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        b[i] = p.B + (size_t)min(n0 + i * 16 + r, p.N - 1) * p.ldb + c * 16;
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto step = [&](auto n_, int kb) {      // n blocks W apart, all their loads first
        constexpr int U = decltype(n_)::value;
        i32x8 fb[U][NT], fa[U][MT];
        unsigned xa[U][MT], xb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = kb + u * W;
#pragma unroll
            for (int i = 0; i < NT; ++i) fb[u][i] = frag_global(b[i] + (size_t)k * 128);
            xb[u] = *reinterpret_cast<const unsigned*>(sb + (k & ~3)) >> ((k & 3) * 8);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int k = kb + u * W;
                if constexpr (AT == A_FP8) {
                    fa[u][j] = frag_global(a[j] + (size_t)k * 128);
                    xa[u][j] = sa[j][k];
                } else fa[u][j] = frag_quantised<AT>(a[j], k, c, p.Ka, xa[u][j]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = mfma_fp8(fb[u][i], fa[u][j], acc[i][j], (int)xb[u], (int)xa[u][j]);
    };
    constexpr int U = MT * NT > 2 || AT != A_FP8 ? 2 : 4;
    int kb = wave;
    for (; kb + (U - 1) * W < nkb; kb += U * W) step(std::integral_constant<int, U>{}, kb);
    for (; kb < nkb; kb += W) step(std::integral_constant<int, 1>{}, kb);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) part[(wave * NT * MT + i * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int t = threadIdx.x; t < NT * MT * 64; t += blockDim.x) {
        f32x4 v = part[t];
        for (int w = 1; w < W; ++w) v += part[w * NT * MT * 64 + t];
        const int l = t & 63, i = (t >> 6) / MT, j = (t >> 6) % MT;
        store_out4(p, m0 + j * 16 + (l & 15), n0 + i * 16 + (l >> 4) * 4, v, gran);
    }
}

__device__ __forceinline__ void glds4(const void* gsrc, void* lds_wave_base) {
    __builtin_amdgcn_global_load_lds(GLB_PTR(gsrc), LDS_PTR(lds_wave_base), 4, 0, 0);
}
template <int N> __device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N > 63 ? 63 : N) : "memory");
}

// ------------------------------------------------------------------------------------------------
// Products too small to fill the chip with 256 x 256 tiles: 64 x 64 tiles, 4 waves (2 x 2, 32 x 32 each), a ring of three K-tiles
// of one block (128 bytes a row, the image of the large kernel), two of them in flight, one barrier per K-tile, three workgroups a
// CU.  The scale words (64 rows of A, then the tile's one block of B) ride in a 1-KiB slot beside each K-tile.  What bounds it is
// the CU's path to the caches (16 KiB a K-tile at about 24 bytes a clock), not the depth of the ring: rings of 2, 4 and 6 and tiles
// of 128 x 64, 64 x 128, 128 x 128, 64 x 32, 32 x 64 and 32 x 32 measured within 10 % or slower over 28 shapes (4020 x 768 x 768:
// 8.4 us, 1000 x 2304 x 2304: 14.6).  Tiles of 128 x 128 whose LDS reads run under the products gain only where 128 to 256 of them fill the
// chip just once (1024 x 4096 x 4096 29 us against 36; 2048 x 2304 x 2304 30 against 23), with two workgroups a CU the other way round
// (30 and 20.6): not kept.  splits > 1: workgroup (tile, s) takes the s-th part of the depth.
//
// AT: e4m3 rows, or 16- / 32-bit rows (p.sa unused, p.lda in bytes, p.Ka columns) that are quantised on their way into LDS: four
// threads a row, their pieces of 8 columns side by side, loaded a K-tile ahead; two slots of A's image and scales behind B's ring.
// A K-tile takes 0.78 us there, what its steps take one behind the other, or 1.8 ns x tiles; GPU time of 201 x 768 x 768 6.6 us, with the
// row quantiser before the product 6.9.  Loads two K-tiles ahead measured the same (hipcc waits for all loads when LDS-DMA is in flight).
// ------------------------------------------------------------------------------------------------
// Tile number lid: groups of `group` columns of tiles one after the other, row by row inside a group (see group_of).
__device__ __forceinline__ void tile_of(int lid, int tiles_m, int tiles_n, int group, int& tm, int& tn) {
    const int per = tiles_m * group, g = lid / per, rem = lid - g * per, w = min(group, tiles_n - g * group);
    tm = rem / w;
    tn = g * group + (rem - tm * w);
}
template <int AT> struct Tile64 {
    static constexpr bool Q = AT != A_FP8;
    static constexpr int SLOTS = 3, IMAGE = (Q ? 64 : 128) * 128, STAGE = IMAGE + 1024, OPS = Q ? 3 : 5;      // LDS-DMA operations a wave and K-tile
    static constexpr int A_SLOT = 64 * 128 + 256, LDS = SLOTS * STAGE + (Q ? 2 * A_SLOT : 0);
};
template <int AT>
__global__ __launch_bounds__(256) void gemm_fp8_tile_kernel(Fp8Args p, int gran, int splits, float* ws, int group) {
    typedef Tile64<AT> T;
    constexpr bool Q = T::Q;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1, nkb = p.K >> 7;
    const int bid = xcd_remap(blockIdx.x, gridDim.x), lid = bid / splits, sp = bid - lid * splits;
    int tm, tn;
    tile_of(lid, (p.M + 63) / 64, (p.N + 63) / 64, group, tm, tn);
    const int m0 = tm * 64, n0 = tn * 64;
    const int kb0 = (int)((int64_t)nkb * sp / splits), nk = (int)((int64_t)nkb * (sp + 1) / splits) - kb0;      // >= 1: splits <= nkb
    // 16-byte pieces: wave w's i-th instruction moves rows 8 (4 i + w) .. + 7 of the [A; B] image
    const unsigned char* src[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = (i * 4 + wave) * 8 + (lane >> 3), chunk = ((lane & 7) ^ ((row >> 1) & 7)) << 4;
        src[i] = (row < 64 ? p.A + (size_t)min(m0 + row, p.M - 1) * p.lda : p.B + (size_t)min(n0 + row - 64, p.N - 1) * p.ldb) + chunk;
    }
    const unsigned char* ssrc = !Q && tid < 64 ? p.sa + (size_t)min(m0 + tid, p.M - 1) * p.lsa : p.sb + (size_t)(n0 >> 7) * p.lsb;
    auto issue = [&](int k, int slot) {
        char* b = smem + slot * T::STAGE;
        constexpr int I0 = Q ? 2 : 0;
#pragma unroll
        for (int i = I0; i < 4; ++i) glds16(src[i] + (size_t)(kb0 + k) * 128, b + ((i - I0) * 4 + wave) * 1024);
        glds4(ssrc + ((kb0 + k) & ~3), b + T::IMAGE + wave * 256);
    };
    const int qrow = tid >> 2, qpiece = tid & 3;
    const unsigned char* arow = p.A + (size_t)min(m0 + qrow, p.M - 1) * p.lda;
    Eight<AT> raw[4];
    auto load_a = [&](int k) {
        if constexpr (Q) {
            const int col = (kb0 + k) * 128 + qpiece * 8;
            if ((kb0 + k) * 128 + 128 <= p.Ka) {      // (the same for all: no branch per piece but in the last block)
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[i].load(arow, col + i * 32, 8);
            } else
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[i].load(arow, col + i * 32, p.Ka - col - i * 32);
        }
    };
    auto quantise_a = [&](int k) {
        if constexpr (Q) {
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = raw[i].grow(m);
            m = Eight<AT>::amax(m);
            m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true));      // lanes 1 and 2 apart: the row's four
            m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, true));
            const unsigned byte = scale_byte(m), slot = lds_addr(smem) + T::SLOTS * T::STAGE + (k & 1) * T::A_SLOT;
            const bool finite = m < 0x7f800000u;
            // (inline asm: before a write it can see hipcc may wait for the LDS-DMA in flight)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int piece = i * 4 + qpiece;
                const u32x2 v = {raw[i].pack(0, byte, finite), raw[i].pack(1, byte, finite)};
                asm volatile("ds_write_b64 %0, %1" ::"v"(slot + qrow * 128 + (((piece >> 1) ^ ((qrow >> 1) & 7)) << 4) + (piece & 1) * 8), "v"(v) : "memory");
            }
            if (qpiece == 0) asm volatile("ds_write_b32 %0, %1" ::"v"(slot + 64 * 128 + qrow * 4), "v"(byte) : "memory");
        }
    };
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int fsw = (r >> 1) & 7;
    const unsigned lds0 = lds_addr(smem), off0 = r * 128 + ((c ^ fsw) << 4), off1 = r * 128 + (((4 + c) ^ fsw) << 4);
    load_a(0);
    issue(0, 0);
    quantise_a(0);
    if (nk > 1) {
        load_a(1);
        issue(1, 1);
    }
    int slot = 0;
    for (int k = 0; k < nk; ++k) {
        if (k + 1 < nk) wait_vm<T::OPS>(); else wait_vm<0>();      // K-tile k has landed (this wave's share), k + 1 stays in flight
        if constexpr (Q) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        phase_barrier();                                             // ... every wave's share; and K-tile k - 1 has been read by all
        if (k + 1 < nk) quantise_a(k + 1);
        if (k + 2 < nk) {
            load_a(k + 2);
            issue(k + 2, slot == 0 ? 2 : slot - 1);
        }
        const unsigned b = lds0 + slot * T::STAGE, as = Q ? lds0 + T::SLOTS * T::STAGE + (k & 1) * T::A_SLOT : b;
        const unsigned ab = as + wm * 4096, bb = b + (Q ? 0 : 8192) + wn * 4096, sc = b + T::IMAGE, asc = Q ? as + 64 * 128 : sc;
        const unsigned a0 = ab + off0, a1 = ab + off1, b0 = bb + off0, b1 = bb + off1;
        u32x4 fa[2][2], fb[2][2];
        unsigned sa[2], sb;
        // (inline asm, reads and wait in one statement: hipcc would wait for every LDS-DMA in flight before a read it can see)
        asm volatile(
            "ds_read_b32 %0, %11 offset:256\n\tds_read_b32 %1, %12\n\tds_read_b32 %2, %12 offset:64\n\t"
            "ds_read_b128 %3, %13\n\tds_read_b128 %4, %14\n\tds_read_b128 %5, %13 offset:2048\n\tds_read_b128 %6, %14 offset:2048\n\t"
            "ds_read_b128 %7, %15\n\tds_read_b128 %8, %16\n\tds_read_b128 %9, %15 offset:2048\n\tds_read_b128 %10, %16 offset:2048\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(sb), "=&v"(sa[0]), "=&v"(sa[1]), "=&v"(fa[0][0]), "=&v"(fa[0][1]), "=&v"(fa[1][0]), "=&v"(fa[1][1]), "=&v"(fb[0][0]),
              "=&v"(fb[0][1]), "=&v"(fb[1][0]), "=&v"(fb[1][1])
            : "v"(sc), "v"(asc + (wm * 32 + r) * 4), "v"(a0), "v"(a1), "v"(b0), "v"(b1)
            : "memory");
        const int sh = ((kb0 + k) & 3) * 8, sha = Q ? 0 : sh;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = mfma_fp8(join8(fb[j][0], fb[j][1]), join8(fa[i][0], fa[i][1]), acc[i][j], (int)(sb >> sh), (int)(sa[i] >> sha));
        slot = slot == 2 ? 0 : slot + 1;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int m = m0 + wm * 32 + i * 16 + r, n = n0 + wn * 32 + j * 16 + c * 4;
            if (splits == 1) store_out4(p, m, n, acc[i][j], gran);
            else if (m < p.M && n < p.N) *reinterpret_cast<f32x4*>(ws + ((size_t)sp * p.M + m) * ((p.N + 3) & ~3) + n) = acc[i][j];
        }
}

// the partial sums of a split product, in the splits' order
__global__ __launch_bounds__(256) void gemm_fp8_join_kernel(Fp8Args p, int gran, int splits, const float* ws) {
    const int n4 = (p.N + 3) >> 2;
    const int64_t all = (int64_t)p.M * n4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / n4), n = (int)(i - (int64_t)m * n4) * 4;
        f32x4 v = reinterpret_cast<const f32x4*>(ws)[i];
        for (int s = 1; s < splits; ++s) v += reinterpret_cast<const f32x4*>(ws)[i + s * all];
        store_out4(p, m, n, v, gran);
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
//
// Measured (warm, 3 operands in rotation): 8192^3 407 us (2.70 PFLOP/s; the library's product with one scale per tensor 410),
// 16384 x 4096 x 4096 206 us (2.66), 51456 x 2304 x 768 99 us (1.85).  What bounds it is the CU's one path to the caches, 64 KiB a
// K-tile in and the tile out, at 16 - 20 bytes a clock (counters: matrix units 65 % busy at 8192^3, LDS 26 %, bank conflicts 2 %):
// 51456 x 2304 x 768 carries 948 MB over it.  Tried without gain: wave priorities around the matrix instructions, reads before the
// next half-tile's issue, two launches of different tile height against the partial last round, other tile orders, a K order turned
// per XCD; a strip of B resident in LDS with rows of A streamed past it (115 us against 112, with a quarter less operand traffic).
// The output costs 16 - 24 of the 100 us at 51456 x 2304 (without its stores K = 256 / 768 / 1536 take 47 / 90 / 160 us, with them 71 /
// 106 / 179, and the same when they all go to 4 MB, so memory is not it: the CU's path again, a fill of that size takes 30).  They leave
// as whole 128-byte lines through LDS, past the cache: through it 110 -> 116; exchanged between lanes by v_permlane16_swap instead,
// in half lines, 100 -> 116.
// ------------------------------------------------------------------------------------------------
#define F8_SCALES 131072
#define F8_BIAS (F8_SCALES + 2 * 2048)
#define F8_STAGE (F8_BIAS + 2048)
#define F8_LDS (F8_STAGE + 8 * 2048)

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

// RB: 16-row blocks of each wave's second 64-row half that are real output (4, 3, 2: tiles of 256, 224, 192 rows).
// GR: columns of an output row stored at once (8 where rows start on 16 bytes and N % 8 == 0; 2; 1).
template <int RB, int GR>
__global__ __launch_bounds__(512, 2) void gemm_fp8_256p_kernel(Fp8Args p, int ntiles, int group_n) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = 128 + 32 * RB, HW = BM / 2, E = 16 / GR * (4 + RB);
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
                if constexpr (GR == 8) st_b128<true>(d[ps], (m < mend && n < p.N) ? off : OOB_OFF, rs);
                else
#pragma unroll
                    for (int j = 0; j < 8; j += GR) {
                        const unsigned o = (m < mend && n + j < p.N) ? off + 2 * j : OOB_OFF;
                        const unsigned v = d[ps][j >> 1];
                        if (GR == 2) asm volatile("buffer_store_dword %0, %1, %2, 0 offen\n\ts_nop 1" ::"v"(v), "v"(o), "s"(rs) : "memory");
                        else if (j & 1) asm volatile("buffer_store_short_d16_hi %0, %1, %2, 0 offen\n\ts_nop 1" ::"v"(v), "v"(o), "s"(rs) : "memory");
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

// More than 64 KiB of dynamic LDS has to be allowed for, once on every GPU that runs the kernel.
template <typename F> static int allow_lds(F kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) dev = 0;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return GETMI_OK;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        getmi_set_error("gemm_fp8: %d bytes of LDS refused: %s", bytes, hipGetErrorString(e));
        return GETMI_ERR_LAUNCH;
    }
    done.fetch_or(bit, std::memory_order_relaxed);
    return GETMI_OK;
}

template <int RB, int GR> static int launch_256p(const Fp8Args& p, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_lds(gemm_fp8_256p_kernel<RB, GR>, F8_LDS, done)) return rc;
    constexpr int BM = 128 + 32 * RB;
    const int ntiles = ((p.M + BM - 1) / BM) * ((p.N + 255) / 256), cus = getmi_cu_budget(), grid = ntiles < cus ? ntiles : cus;
    hipLaunchKernelGGL((gemm_fp8_256p_kernel<RB, GR>), dim3(grid), dim3(512), F8_LDS, st, p, ntiles, pick_group(p.M, p.N, p.K, BM, grid));
    GETMI_CHECK_LAUNCH("gemm_fp8");
    return GETMI_OK;
}
template <int MT, int NT, int AT = A_FP8> static int launch_rows(const Fp8Args& p, int gran, hipStream_t st) {
    const int nkb = p.K / 128, wgs = ((p.N + 16 * NT - 1) / (16 * NT)) * ((p.M + 16 * MT - 1) / (16 * MT));
    const int W = nkb >= 32 && wgs <= 256 ? 16 : nkb >= 16 ? 8 : 4;      // 4, 8 and 16 measure alike where either applies
    GETMI_CHECK_ARG((int64_t)wgs * W * 64 < (int64_t)1 << 32, "gemm_fp8: N=%d too large", p.N);      // a launch is at most 2^32 - 1 threads wide
    hipLaunchKernelGGL((gemm_fp8_rows_kernel<MT, NT, AT>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT)), dim3(64 * W),
                       (size_t)W * MT * NT * 1024, st, p, gran);
    GETMI_CHECK_LAUNCH("gemm_fp8");
    return GETMI_OK;
}
// Columns of 64 x 64 tiles in a group: the tiles that run at once on an XCD (3 on each of 32 CUs) make a square of the output, so that
// its L2 fetches the fewest rows of both operands.  Against whole rows of tiles: 1024 x 4096 x 4096 43 -> 36 us, 256 x 8192 x 8192 41.6 ->
// 35.6, 400 x 3000 x 3000 15.4 -> 12.7.
static int group_of(int M, int N, int splits) {
    const int tm = (M + 63) / 64, tn = (N + 63) / 64;
    int64_t t = ((int64_t)tm * tn + 7) / 8;
    if (t > 96 / splits) t = 96 / splits;
    int g = 1;
    while (g * g < t) ++g;
    if ((int64_t)g * tm < t) g = (int)((t + tm - 1) / tm);
    return g < tn ? g : tn;
}
template <int AT = A_FP8> static int launch_tile(const Fp8Args& p, int gran, int splits, float* ws, hipStream_t st) {
    const int64_t tiles = (int64_t)((p.M + 63) / 64) * ((p.N + 63) / 64);
    GETMI_CHECK_ARG(tiles * splits < 1 << 24, "gemm_fp8: M=%d N=%d too large", p.M, p.N);      // a launch is at most 2^32 - 1 threads wide
    hipLaunchKernelGGL(gemm_fp8_tile_kernel<AT>, dim3((unsigned)(tiles * splits)), dim3(256), Tile64<AT>::LDS, st, p, gran, splits, ws,
                       group_of(p.M, p.N, splits));
    if (splits > 1) {
        const int64_t blocks = ((int64_t)p.M * ((p.N + 3) / 4) + 255) / 256;
        hipLaunchKernelGGL(gemm_fp8_join_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, p, gran, splits,
                           (const float*)ws);
    }
    GETMI_CHECK_LAUNCH("gemm_fp8");
    return GETMI_OK;
}

// What a launch takes, in us (see plan_of): 64 x 64 tiles; a round of 256 / 224 / 192-row tiles on the part `fill` of the CUs.
static double tile_time(int M, int N, int nk) {
    const double t = (double)((M + 63) / 64) * ((N + 63) / 64) * 1.1e-3;
    return 2.5 + nk * (t > 0.34 ? t : 0.34);
}
static double round_time(int rb, int nk, double fill) {
    return (nk * (1.15 + 0.7 * fill) + 3.5) * (rb == 4 ? 1.0 : rb == 3 ? 0.93 : 0.87);
}

template <int GR> static int launch_256p(const Fp8Args& p, int rb, hipStream_t st) {
    return rb == 4 ? launch_256p<4, GR>(p, st) : rb == 3 ? launch_256p<3, GR>(p, st) : launch_256p<2, GR>(p, st);
}
// Tile height: the one whose rounds take least.  Where the last round would hold very few tiles, whole rounds only, and the rows
// behind them go to 64 x 64 tiles in a second launch (charged twice: alone on the chip they run at half their rate).  51456 x 2304 x
// 768, 7.07 rounds: 113 -> 109 us; 33000 x 512 x 4096, 1.01 rounds: 90 -> 74; at 2.25 rounds of 6000^3 it would cost 195 -> 218.
template <int GR> static int launch_big(const Fp8Args& p, int gran, hipStream_t st) {
    const int cus = getmi_cu_budget(), tn = (p.N + 255) / 256, nk = p.K >> 7;
    int best = 4, rows = p.M;
    double cost = 0;
    for (int rb = 4; rb >= 2; --rb) {
        const int bm = 128 + 32 * rb;
        const int64_t tiles = (int64_t)((p.M + bm - 1) / bm) * tn, before = (tiles - 1) / cus;      // whole rounds before the last
        const double most = before * round_time(rb, nk, 1.0), whole = most + round_time(rb, nk, (double)(tiles - before * cus) / cus);
        if (cost == 0 || whole < cost - 1e-9) { cost = whole; best = rb; rows = p.M; }
        const int64_t cut = before * cus / tn * bm;
        if (cut > 0 && cut < p.M) {
            const double c = most + 2.0 * tile_time((int)(p.M - cut), p.N, nk);
            if (c < cost - 1e-9) { cost = c; best = rb; rows = (int)cut; }
        }
    }
    Fp8Args q = p;
    q.M = rows;
    if (const int rc = launch_256p<GR>(q, best, st)) return rc;
    if (rows == p.M) return GETMI_OK;
    q.A += (size_t)rows * p.lda; q.sa += (size_t)rows * p.lsa; q.out += (size_t)rows * p.ldo; q.M = p.M - rows;
    return launch_tile(q, gran, 1, nullptr, st);
}

// Which kernel takes a product: by its shape alone.  Both sides measured on MI355X (us, back to back, operands in rotation):
//   up to 16 rows    rows kernel: 1 x 8192 x 8192 13.6 (4.9 TB/s) against 64-row tiles 22.5; 8 x 768 x 8192 9.0 against 21.7.  Two
//                    16-row groups of B a workgroup where both sides are wide (16 x 8192 x 8192 20.0 -> 17.2; 1 row: 13.6 -> 16.6)
//   up to 32, N <= 4096   rows kernel with two row groups: 8 x 768 x 8192 9.8; at N = 8192 64-row tiles in two splits win, 22 -> 15.6
//   64 x 64 tiles    a K-tile costs a CU 16 KiB of its one path to the caches (1.0 - 1.2 ns x tiles over the chip), a lone workgroup 0.34 us
//   256 x 256 tiles  1.15 us a K-tile with few CUs busy, 1.85 with all (the same path: 64 KiB), 3.5 for the tile's ends
//                    4020 x 768 x 768 8.6 against 12.2, 12060 x 768 x 768 18.3 against 13.3, 2000 x 4096 x 4096 76 against 39
//   depth of 6144 on and few 64-row tiles: the depth is split and joined by a second kernel (64 x 8192 x 8192 23.5 -> 17.1,
//                    300 x 768 x 8192 22.9 -> 13.1; at 4096 x 4096 the join costs what it saves: 13.1 -> 13.3)
enum { ROWS11, ROWS12, ROWS21, TILE, BIG };
struct Plan { int kind, splits; };
static Plan plan_of(int M, int N, int K) {
    if (M <= 16) return Plan{M > 8 && N >= 8192 ? ROWS12 : ROWS11, 1};
    if (M <= 32 && N <= 4096) return Plan{ROWS21, 1};
    const int nk = K >> 7;
    const double t64 = (double)((M + 63) / 64) * ((N + 63) / 64), t256 = (double)((M + 255) / 256) * ((N + 255) / 256);
    const double small = tile_time(M, N, nk);
    const double rounds = (double)(((int64_t)t256 + 255) / 256);
    const double large = 2.0 + rounds * (nk * (1.15 + 0.7 * (t256 < 256 ? t256 / 256 : 1.0)) + 3.5);
    if (nk >= 2 && large < small) return Plan{BIG, 1};
    return Plan{TILE, nk >= 48 && t64 <= 128 ? (t64 <= 64 ? 4 : 2) : 1};
}
size_t getmi_gemm_fp8_workspace_bytes_impl(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fff0000 || N > 0x7fff0000) return 0;
    const Plan pl = plan_of(M, N, K);
    return pl.splits == 1 ? 0 : (size_t)pl.splits * M * ((N + 3) & ~3) * sizeof(float);
}
static int granularity(const void* out, int N, int64_t ldo) {
    const uint64_t all = (uintptr_t)out / 2 | (uint64_t)N | (uint64_t)ldo;
    return all % 8 == 0 && (uintptr_t)out % 16 == 0 ? 8 : all % 4 == 0 && (uintptr_t)out % 8 == 0 ? 4 : all % 2 == 0 && (uintptr_t)out % 4 == 0 ? 2 : 1;
}

int getmi_gemm_fp8_impl(const void* A, const void* sa, const void* B, const void* sb, const float* bias, void* out, int M, int N, int K,
                        int64_t lda, int64_t ldb, int64_t ldo, int lsa, int lsb, void* workspace, size_t workspace_bytes, hipStream_t st) {
    GETMI_CHECK_ARG(M >= 0 && N >= 0 && M <= 0x7fff0000 && N <= 0x7fff0000 && K > 0 && K <= 0x7fff0000 && K % 128 == 0, "gemm_fp8: M=%d N=%d K=%d (K is a multiple of 128: pad with zeros)", M, N, K);
    if (M == 0 || N == 0) return GETMI_OK;
    GETMI_CHECK_ARG(A && sa && B && sb && out && (uintptr_t)out % 2 == 0, "gemm_fp8: null or odd pointer");
    GETMI_CHECK_ARG(((uintptr_t)A | (uintptr_t)B | (uint64_t)lda | (uint64_t)ldb) % 16 == 0 && lda >= 0 && ldb >= 0 && ldo >= N,
                    "gemm_fp8: operand rows have to start on 16 bytes, output rows must not overlap");
    GETMI_CHECK_ARG(((uintptr_t)sa | (uintptr_t)sb | (unsigned)lsa | (unsigned)lsb) % 4 == 0 && lsa >= 0 && lsb >= 0,
                    "gemm_fp8: scale rows have to start on 4 bytes");
    Fp8Args p{(const unsigned char*)A, (const unsigned char*)sa, (const unsigned char*)B, (const unsigned char*)sb, bias, (bf16_t*)out,
              (size_t)lda, (size_t)ldb, (size_t)ldo, lsa, lsb, M, N, K, K};
    const int gran = granularity(out, N, ldo);
    const Plan pl = plan_of(M, N, K);
    GETMI_CHECK_ARG(pl.splits == 1 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= getmi_gemm_fp8_workspace_bytes_impl(M, N, K)),
                    "gemm_fp8: workspace of getmi_gemm_fp8_workspace_bytes(M, N, K) needed");
    if (pl.kind == ROWS11) return launch_rows<1, 1>(p, gran, st);
    if (pl.kind == ROWS12) return launch_rows<1, 2>(p, gran, st);
    if (pl.kind == ROWS21) return launch_rows<2, 1>(p, gran, st);
    // The large kernel addresses each operand with 32 bits: more rows than that reaches go in several launches (1000000 x 2304 x 768,
    // 4.6 GB of output: 2076 us, against 4281 with 64 x 64 tiles).
    const size_t lim = 0xF0000000ull - (size_t)K;
    auto reach = [&](size_t ld) { return ld ? lim / ld : (size_t)M; };
    size_t most = std::min(std::min(reach(p.lda), reach(p.ldo * 2)), std::min(reach(lsa), (size_t)M));
    if (most < (size_t)M) most &= ~(size_t)255;
    if (pl.kind == BIG && (most == (size_t)M || most >= 4096) && (size_t)N <= std::min(reach(p.ldb), reach(lsb))) {
        const int64_t parts = (M + (int64_t)most - 1) / (int64_t)most, per = parts == 1 ? M : ((M + parts - 1) / parts + 255) & ~(int64_t)255;
        for (int64_t m = 0; m < M; m += per) {
            Fp8Args q = p;
            q.A += m * p.lda; q.sa += m * lsa; q.out += m * p.ldo; q.M = (int)std::min(per, M - m);
            if (const int rc = gran == 8 ? launch_big<8>(q, gran, st) : gran >= 2 ? launch_big<2>(q, gran, st) : launch_big<1>(q, gran, st)) return rc;
        }
        return GETMI_OK;
    }
    return launch_tile(p, gran, pl.splits, (float*)workspace, st);
}

// Up to 16 rows of fp32 / bf16, quantised inside the product: x[M, K] (rows ldx elements apart), B[N, Kp] and its scales as above.
int getmi_linear_fp8_rows_impl(const void* x, int xt, int64_t ldx, const void* B, const void* sb, const float* bias, void* out, int M, int N,
                               int K, int64_t ldb, int64_t ldo, int lsb, hipStream_t st) {
    GETMI_CHECK_ARG(M >= 0 && M <= 16 && N >= 0 && N <= 0x7fff0000 && K > 0 && K <= 0x7fff0000, "linear_fp8_rows: M=%d N=%d K=%d (M <= 16)", M, N, K);
    if (M == 0 || N == 0) return GETMI_OK;
    GETMI_CHECK_ARG(x && B && sb && out && (uintptr_t)out % 2 == 0 && (xt == A_F32 || xt == A_BF16), "linear_fp8_rows: null or odd pointer, or type");
    GETMI_CHECK_ARG(((uintptr_t)B | (uint64_t)ldb) % 16 == 0 && ldb >= 0 && ldx >= 0 && ldo >= N, "linear_fp8_rows: weight rows have to start on 16 bytes, output rows must not overlap");
    GETMI_CHECK_ARG(((uintptr_t)sb | (unsigned)lsb) % 4 == 0 && lsb >= 0, "linear_fp8_rows: scale rows have to start on 4 bytes");
    const int Kp = (K + 127) / 128 * 128, gran = granularity(out, N, ldo);
    Fp8Args p{(const unsigned char*)x, nullptr, (const unsigned char*)B, (const unsigned char*)sb, bias, (bf16_t*)out,
              (size_t)ldx * (xt == A_F32 ? 4 : 2), (size_t)ldb, (size_t)ldo, 0, lsb, M, N, Kp, K};
    return xt == A_F32 ? launch_rows<1, 1, A_F32>(p, gran, st) : launch_rows<1, 1, A_BF16>(p, gran, st);
}

// Any number of rows of fp32 / bf16, quantised inside the product by every 64 x 64 tile that reads them.
int getmi_linear_fp8_tiles_impl(const void* x, int xt, int64_t ldx, const void* B, const void* sb, const float* bias, void* out, int M, int N,
                                int K, int64_t ldb, int64_t ldo, int lsb, hipStream_t st) {
    GETMI_CHECK_ARG(M >= 0 && M <= 0x7fff0000 && N >= 0 && N <= 0x7fff0000 && K > 0 && K <= 0x7fff0000, "linear_fp8_tiles: M=%d N=%d K=%d", M, N, K);
    if (M == 0 || N == 0) return GETMI_OK;
    GETMI_CHECK_ARG(x && B && sb && out && (uintptr_t)out % 2 == 0 && (xt == A_F32 || xt == A_BF16), "linear_fp8_tiles: null or odd pointer, or type");
    GETMI_CHECK_ARG(((uintptr_t)B | (uint64_t)ldb) % 16 == 0 && ldb >= 0 && ldx >= 0 && ldo >= N, "linear_fp8_tiles: weight rows have to start on 16 bytes, output rows must not overlap");
    GETMI_CHECK_ARG(((uintptr_t)sb | (unsigned)lsb) % 4 == 0 && lsb >= 0, "linear_fp8_tiles: scale rows have to start on 4 bytes");
    const int Kp = (K + 127) / 128 * 128, gran = granularity(out, N, ldo);
    Fp8Args p{(const unsigned char*)x, nullptr, (const unsigned char*)B, (const unsigned char*)sb, bias, (bf16_t*)out,
              (size_t)ldx * (xt == A_F32 ? 4 : 2), (size_t)ldb, (size_t)ldo, 0, lsb, M, N, Kp, K};
    return xt == A_F32 ? launch_tile<A_F32>(p, gran, 1, nullptr, st) : launch_tile<A_BF16>(p, gran, 1, nullptr, st);
}
