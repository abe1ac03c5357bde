// Tiles of the MFMA products (gemm.hip, act8.hip): operand images in LDS, fragment reads, the persistent grid's work items and
// the pieces of the phased 256x256 kernels.  Device code shared by translation units; see gemm.hip for the structure.
#pragma once
#include "common.h"

namespace {

constexpr int BK = 64;

// Tile configurations.
//   small:  128x128 output tile, 4 waves (2x2, 64x64 per wave), one LDS buffer, two barriers per K step;
//           three workgroups per CU hide the staging latency.  Small outputs (decoder, ragged shapes).
//   tiny:   64x64 output tile, otherwise as small: outputs too small to give every CU a 128x128 tile
//           (the decoder's 2-token sequences).
//   phased: 256x256 output tile, 8 waves (2x4), one workgroup per CU, all 160 KiB of LDS as a ring of
//           half-tiles; see the kernel below.  moff/noff give the tile-relative origin of a wave's
//           i-th / j-th 16x16 accumulator block.
}  // namespace
struct CfgSmall {
    static constexpr int BM = 128, BN = 128, WGM = 2, WGN = 2, MI = 4, NJ = 4;
    static constexpr __device__ __forceinline__ int moff(int wm, int i) { return wm * 64 + i * 16; }
    static constexpr __device__ __forceinline__ int noff(int wn, int j) { return wn * 64 + j * 16; }
};
// small8: the 128x128 tile with eight waves of 32x64: two waves to a SIMD, so that one's fragment reads run under the other's
//           MFMAs where a CU has a single tile (linear_ce.hip's mid-sized products).  64 columns a wave, as in the small tile.
struct CfgSmall8 {
    static constexpr int BM = 128, BN = 128, WGM = 4, WGN = 2, MI = 2, NJ = 4;
    static constexpr __device__ __forceinline__ int moff(int wm, int i) { return wm * 32 + i * 16; }
    static constexpr __device__ __forceinline__ int noff(int wn, int j) { return wn * 64 + j * 16; }
};
struct CfgTiny {
    static constexpr int BM = 64, BN = 64, WGM = 2, WGN = 2, MI = 2, NJ = 2;
    static constexpr __device__ __forceinline__ int moff(int wm, int i) { return wm * 32 + i * 16; }
    static constexpr __device__ __forceinline__ int noff(int wn, int j) { return wn * 32 + j * 16; }
};
struct CfgPhased {
    static constexpr int BM = 256, BN = 256, WGM = 2, WGN = 4, MI = 8, NJ = 4;
    static constexpr __device__ __forceinline__ int moff(int wm, int i) { return (i >> 2) * 128 + wm * 64 + (i & 3) * 16; }
    static constexpr __device__ __forceinline__ int noff(int wn, int j) { return wn * 64 + j * 16; }   // B halves interleave 32-column blocks
};
namespace {

// Per-lane source offset (bytes, relative to the tile's first row / column) of the 16-byte chunk
// that lands at lane-linear LDS position g (16-byte units) of a tile image.
//   K-contiguous operand : image [ROWS][64] bf16, 128-byte rows; chunk c of row r sits at c ^ ((r>>1)&7).
//   K-strided operand    : image [64][ROWS] bf16; the 32-byte unit u of k-row k sits at u ^ h(k),
//                          h(k) = (k&3) | ((k>>3)&1)<<2, masked to the units a k-row has
//                          (conflict-free ds_read_b64_tr_b16 from 128 rows up).
// With SPLIT (the phased kernel's B halves) image row r of a half is tile row (r>>5)*64 + (r&31): a
// half holds one 32-row block out of every 64 rows, so that a wave's two 32-row slices (one per half)
// are 64 CONSECUTIVE tile rows.
template <bool TRANS, int ROWS, bool SPLIT = false>
__device__ __forceinline__ uint32_t stage_offset(int g, int ld, long long heads = 0) {
    if (!TRANS) {
        const int r = g >> 3, cs = g & 7;
        const int c = cs ^ ((r >> 1) & 7);
        const int rs = SPLIT ? ((r >> 5) * 64 + (r & 31)) : r;
        return (uint32_t)(rs * ld + c * 8) * 2u;
    } else {
        constexpr int CPR = ROWS / 8;                 // 16-byte chunks per k-row
        const int k = g / CPR, cs = g % CPR;
        const int hk = ((k & 3) | (((k >> 3) & 1) << 2)) & (ROWS / 16 - 1);
        const int c = (((cs >> 1) ^ hk) << 1) | (cs & 1);
        const int csrc = SPLIT ? ((c >> 2) * 8 + (c & 3)) : c;
        if (heads) return (uint32_t)(((csrc >> 3) * heads + k * 64 + (csrc & 7) * 8) * 2);      // head-major: 8 chunks per head
        return (uint32_t)(k * ld + csrc * 8) * 2u;
    }
}

// 16 rows x 32 k fragment (one v_mfma_f32_16x16x32_bf16 operand) for rows rb..rb+15, k-step kk.
// With RAW_ASM the transposed reads are issued as inline assembly: the compiler then neither waits
// for them (the caller must s_waitcnt lgkmcnt before the first use) nor drains every LDS-DMA in flight
// ahead of them, which it does for the builtin (it cannot tell that the DMA targets another slot).
template <bool TRANS, int ROWS, bool RAW_ASM = false>
__device__ __forceinline__ bf16x8 read_frag(const char* tile, int rb, int kk, int lane) {
    if (!TRANS) {
        const int row = rb + (lane & 15);
        const int c = kk * 4 + (lane >> 4);
        const int addr = row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
        return *reinterpret_cast<const bf16x8*>(tile + addr);
    } else {
        constexpr int RB = ROWS * 2;                  // bytes per k-row
        const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
        const int u = rb >> 4;
        const int hk = (q | ((g & 1) << 2)) & (ROWS / 16 - 1);
        const int k0 = kk * 32 + 8 * g + q;
        const int addr0 = k0 * RB + ((u ^ hk) << 5) + p * 8;
        bf16x4 lo, hi;
        if (RAW_ASM) {
            const uint32_t a = (uint32_t)(uintptr_t)LDS_PTR(tile + addr0);
            asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(lo) : "v"(a));
            asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(a), "n"(4 * RB));
        } else {
            lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(tile + addr0));
            hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(tile + addr0 + 4 * RB));
        }
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// Item of workgroup b in round `round` of a persistent grid of G workgroups over T items, or -1.
// Within a round the workgroups that share an XCD (equal b % 8) take consecutive items.
__device__ __forceinline__ int item_of(int b, int round, int G, int T) {
    const int first = round * G;
    if (first >= T) return -1;
    const int count = min(G, T - first);
    if (b >= count) return -1;
    return first + xcd_remap(b, count);
}

}  // namespace

// Transposed fragment reads are inline assembly here (see read_frag): wait for all LDS reads of the
// phase before its MFMAs, and keep the scheduler from hoisting anything above the wait.
#define PACED_WAIT_LDS_READS()                                \
    do {                                                      \
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    \
        __builtin_amdgcn_sched_barrier(0);                    \
    } while (0)

// a raw barrier that the instruction scheduler may not move anything across (MFMAs included)
#define PACED_PINNED_BARRIER()                 \
    do {                                       \
        __builtin_amdgcn_sched_barrier(0);     \
        __builtin_amdgcn_s_barrier();          \
        __builtin_amdgcn_sched_barrier(0);     \
    } while (0)

#define PACED_STAGE_HALF(rsrc, dst, off, soff)                                                           \
    do {                                                                                                 \
        __builtin_amdgcn_raw_ptr_buffer_load_lds((rsrc), LDS_PTR((dst)), 16, (off)[0], (soff), 0, 0);         \
        __builtin_amdgcn_raw_ptr_buffer_load_lds((rsrc), LDS_PTR((dst) + 8192), 16, (off)[1], (soff), 0, 0);  \
    } while (0)

namespace {

// Empty volatile asm that "rewrites" the eight accumulators of a quadrant: MFMAs are pure register
// operations, which instruction selection otherwise floats across the barriers into the load sections.
__device__ __forceinline__ void pin_quadrant(f32x4 (&acc)[8][4], int ha, int hb) {
    asm volatile("" : "+v"(acc[ha * 4 + 0][hb * 2 + 0]), "+v"(acc[ha * 4 + 0][hb * 2 + 1]),
                      "+v"(acc[ha * 4 + 1][hb * 2 + 0]), "+v"(acc[ha * 4 + 1][hb * 2 + 1]),
                      "+v"(acc[ha * 4 + 2][hb * 2 + 0]), "+v"(acc[ha * 4 + 2][hb * 2 + 1]),
                      "+v"(acc[ha * 4 + 3][hb * 2 + 0]), "+v"(acc[ha * 4 + 3][hb * 2 + 1]));
}

template <bool NATURAL>
__device__ __forceinline__ void quadrant_mfma(const bf16x8 (&fa)[4][2], const bf16x8 (&fb)[2][2], f32x4 (&acc)[8][4], int ha, int hb) {
    pin_quadrant(acc, ha, hb);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f32x4& c = acc[ha * 4 + i][hb * 2 + j];
                if (NATURAL) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i][kk], fb[j][kk], c, 0, 0, 0);
                else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j][kk], fa[i][kk], c, 0, 0, 0);
            }
    __builtin_amdgcn_s_setprio(0);
    pin_quadrant(acc, ha, hb);
}

__device__ __forceinline__ int ring_wrap(int x) { return x >= 10 ? x - 10 : x; }

}  // namespace
