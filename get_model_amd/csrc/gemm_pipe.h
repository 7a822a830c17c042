// Pieces that the persistent LDS-DMA pipelines share (gemm.hip: bf16, gemm_fp8.hip: e4m3): phase barrier, bounds-checked streamed
// stores, counted waits, the LDS transposition of the epilogue, and the order in which a persistent workgroup walks its output tiles.
#pragma once
#include "common.h"

__device__ __forceinline__ void phase_barrier() {
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
#define OOB_OFF 0xFFFFFFF0u

__device__ __forceinline__ u32x4 make_rsrc(const void* ptr, unsigned bytes) {
    const unsigned long long a = (unsigned long long)ptr;
    return (u32x4){(unsigned)a, (unsigned)(a >> 32) & 0xffffu, bytes, 0x00020000u};
}
__device__ __forceinline__ void st_b64(u32x2 v, unsigned off, u32x4 rs) {
    asm volatile("buffer_store_dwordx2 %0, %1, %2, 0 offen\n\ts_nop 1" ::"v"(v), "v"(off), "s"(rs) : "memory");
}
template <bool NT = false>
__device__ __forceinline__ void st_b128(u32x4 v, unsigned off, u32x4 rs) {
    if constexpr (NT) asm volatile("buffer_store_dwordx4 %0, %1, %2, 0 offen nt\n\ts_nop 1" ::"v"(v), "v"(off), "s"(rs) : "memory");
    else asm volatile("buffer_store_dwordx4 %0, %1, %2, 0 offen\n\ts_nop 1" ::"v"(v), "v"(off), "s"(rs) : "memory");
}

// wait until at most 2*halftiles (+ EXTRA) vector-memory operations of this wave are outstanding
template <int EXTRA>
__device__ __forceinline__ void wait_halftiles_x(int halftiles) {
    constexpr int C5 = (10 + EXTRA > 63) ? 63 : 10 + EXTRA, C4 = (8 + EXTRA > 63) ? 63 : 8 + EXTRA,
                  C3 = (6 + EXTRA > 63) ? 63 : 6 + EXTRA, C2 = (4 + EXTRA > 63) ? 63 : 4 + EXTRA,
                  C1 = (2 + EXTRA > 63) ? 63 : 2 + EXTRA, C0 = (EXTRA > 63) ? 63 : EXTRA;
    if (halftiles >= 5) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(C5) : "memory");
    else if (halftiles == 4) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(C4) : "memory");
    else if (halftiles == 3) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(C3) : "memory");
    else if (halftiles == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(C2) : "memory");
    else if (halftiles == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(C1) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"i"(C0) : "memory");
}

// Wave-private LDS transposition of one 16-row x 128-byte block, entirely in inline asm: a compiler-visible access
// to LDS that LDS-DMA also writes makes hipcc drain vmcnt to 0 first.  Writes, wait, reads, wait in ONE statement
// (outputs early-clobber), so no register is reused before the LDS has consumed / produced it.
__device__ __forceinline__ void stage_w64x4_r128x2(unsigned wa, unsigned ra, u32x2 q0, u32x2 q1, u32x2 q2, u32x2 q3,
                                                   u32x4& d0, u32x4& d1) {
    asm volatile(
        "ds_write_b64 %2, %6\n\tds_write_b64 %3, %7\n\tds_write_b64 %4, %8\n\tds_write_b64 %5, %9\n\t"
        "s_waitcnt lgkmcnt(0)\n\t"
        "ds_read_b128 %0, %10\n\tds_read_b128 %1, %10 offset:1024\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(d0), "=&v"(d1)
        : "v"(wa), "v"(wa ^ 32u), "v"(wa ^ 64u), "v"(wa ^ 96u), "v"(q0), "v"(q1), "v"(q2), "v"(q3), "v"(ra)
        : "memory");
}
// Which output tiles a persistent workgroup walks, and in which order.
// Logical tile order = column-group major: the N-tiles are cut into groups of `group_n` columns, and inside a group the
// order is row-block major (tm, then the group's columns).  XCD x (the workgroups with equal blockIdx % 8, made contiguous
// by xcd_remap) takes the x-th EIGHTH of that order for the whole launch, its workgroups striding through it together.
// So at any time the 32 workgroups of an XCD share a few row blocks of A and at most group_n column blocks of B, and
// those B blocks stay in the XCD's 4 MiB L2 from round to round (the host picks group_n so that they fit): with plain
// row-major rounds dealt across the XCDs every XCD re-fetched ALL of B every round (fc1: 12 blocks = 4.7 MB > L2;
// rocprofv3 FETCH_SIZE 448 MB per launch for 84 MB of operands).  group_n == 0 or a grid that is not a multiple of 8:
// the old round-robin order.
struct TileWalk {
    int first, stride, count, tiles_m, tiles_n, group_n;
    __device__ __forceinline__ void init(int bslot, int G, int ntiles, int tm_, int tn_, int gn_) {
        tiles_m = tm_; tiles_n = tn_;
        if (gn_ > 0 && (G & 7) == 0) {
            group_n = gn_;
            const int q = G >> 3, x = bslot / q, c = bslot - x * q;
            const int lo = (int)((long long)ntiles * x / 8), hi = (int)((long long)ntiles * (x + 1) / 8);
            first = lo + c; stride = q; count = (hi - lo - c + q - 1) / q;      // >= 1: hi - lo >= q because ntiles >= G
        } else {
            group_n = tn_;
            first = bslot; stride = G; count = (ntiles - bslot + G - 1) / G;
        }
    }
    // tile i of this workgroup (i clamped to the last one: look-ahead past the end re-stages the last tile, never used)
    __device__ __forceinline__ void decode(int i, int& tm, int& tn) const {
        const int lid = first + min(i, count - 1) * stride;
        const int per = tiles_m * group_n;
        const int cg = lid / per, rem = lid - cg * per;
        const int w = min(group_n, tiles_n - cg * group_n);
        tm = rem / w;
        tn = cg * group_n + (rem - tm * w);
    }
};
