// Activation checkpoints in 8 bits, and the weight gradient that reads them.
//
// A checkpoint of x [T, n] is its e4m3 codes [T, n] and one power-of-two scale (exponent + 127 in a byte) for 32 tokens of a
// feature, [ceil(T/32), n].  Of the 32 values the scale is the smallest power of two, 2^-117 at least, that brings the largest
// magnitude to 448 or less, so no value saturates and scaling is exact; codes round to nearest, ties to even.  With the scale
// 2^120 codes stop at 240 (256 * 2^120 would read back as infinity).  A block that holds a NaN or an infinity is stored as NaNs
// (scale byte 255): it stays visible.  A code has four significant bits and scales stop at 2^-117, so every checkpoint value
// is a bf16 value and reading back rounds nothing.
// Blocks run along the tokens because a weight gradient contracts over tokens: all eight values of a lane's MFMA fragment
// (eight tokens of one feature) share one scale, and v_cvt_scalef32_pk_bf16_fp8 applies it while it converts.
// Writing and reading are bound by memory: 139264 x 768 in 51.5 us (6.3 TB/s) and 55 us (5.9 TB/s).  The gradient is bound by the
// matrix cores where tokens are many: 2304 x 768 from 139264 tokens in 411 to 442 us on different cards, slabs' sum
// included (1.12 to 1.20 PFLOP/s; the bf16 products of gemm.hip reach 1.25 to 1.35 on large squares, the vendor's 1.39);
// 512 x 2048 from 1001 tokens in 8.7 us, by latency.  (A card that was idle takes some sixty launches of the large one to settle: 484 us
// at first, 405 to 427 from then on, and 11 for the slabs' sum.)
#include "gemm_tiles.h"
#include <type_traits>

namespace {

constexpr int QBLOCK = 32;                 // tokens per scale
constexpr int MAX_T = 0x7fffffff - 63;     // tokens of a call: rounded up to K steps they are still an int
constexpr int MIN_CODE = 127 - 117, MAX_CODE = 127 + 120, NAN_CODE = 255;

// ------------------------------------------------------------------------------------------------ writing and reading
// One thread per 32 tokens x 2 features: 32 loads of 4 bytes in flight (256-byte runs of a wave), the maxima in its own
// registers (integer maxima of the magnitudes' bits), no exchange between lanes.  Wider pieces measured slower at every size:
// 139264 x 768 in 51.5 us with 2 features a thread, 54 with 4, 57 with 8; 300 x 512 in 5.2, 5.8 and 7.0 (fewer waves).
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
__global__ void __launch_bounds__(256) act8_quantize_kernel(const bf16* __restrict__ x, int ldx, unsigned char* __restrict__ q,
                                                            unsigned char* __restrict__ scale, int T, int n, int nblk) {
    const int chunks = n >> 1;
    const long long total = (long long)nblk * chunks;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < total; id += (long long)gridDim.x * 256) {
        const int blk = (int)(id / chunks), c = (int)(id - (long long)blk * chunks);
        const int rows = min(QBLOCK, T - blk * QBLOCK);
        const bf16* src = x + (size_t)blk * QBLOCK * ldx + c * 2;
        uint32_t v[QBLOCK];
#pragma unroll
        for (int r = 0; r < QBLOCK; ++r) v[r] = r < rows ? __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(src + (size_t)r * ldx)) : 0u;
        u16x2 top = {};
#pragma unroll
        for (int r = 0; r < QBLOCK; ++r) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[r] & 0x7fff7fffu));
        float inv[2], lim[2];
        uint32_t nan = 0, code = 0;        // codes that make a block NaN, scale bytes
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int bits = top[e];
            int k = (bits >> 7) - 8 + ((bits & 0x7f) > 0x60 ? 1 : 0);        // 448 = 1.75 * 2^8
            k = max(k, MIN_CODE);
            inv[e] = __uint_as_float((uint32_t)(254 - k) << 23);
            lim[e] = k == MAX_CODE ? 240.f : 448.f;
            if (bits >= 0x7f80) { nan |= 0x7fu << (8 * e); k = NAN_CODE; inv[e] = 0.f; }
            code |= (uint32_t)k << (8 * e);
        }
        *reinterpret_cast<unsigned short*>(scale + (size_t)blk * n + c * 2) = (unsigned short)code;
        unsigned char* dst = q + (size_t)blk * QBLOCK * n + c * 2;
#pragma unroll
        for (int r = 0; r < QBLOCK; ++r) {
            const float lo = __uint_as_float(v[r] << 16) * inv[0], hi = __uint_as_float(v[r] & 0xffff0000u) * inv[1];
            const uint32_t o = ((uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(lo, -lim[0], lim[0]),
                                                                           __builtin_amdgcn_fmed3f(hi, -lim[1], lim[1]), 0, false) & 0xffffu) | nan;
            if (r < rows) __builtin_nontemporal_store((unsigned short)o, reinterpret_cast<unsigned short*>(dst + (size_t)r * n));
        }
    }
}

// One thread per 16 tokens x 8 features: a wave stores whole 1 KiB runs (16 features to a thread, two 16-byte stores 32 bytes
// apart: 84 us against 139264 x 768).
constexpr int DQ_ROWS = 16;
__global__ void __launch_bounds__(256) act8_dequantize_kernel(const unsigned char* __restrict__ q, const unsigned char* __restrict__ scale,
                                                              bf16* __restrict__ y, int ldy, int T, int n) {
    const int chunks = n >> 3;
    const long long total = (long long)((T + DQ_ROWS - 1) / DQ_ROWS) * chunks;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < total; id += (long long)gridDim.x * 256) {
        const int tb = (int)(id / chunks), c = (int)(id - (long long)tb * chunks);
        const int rows = min(DQ_ROWS, T - tb * DQ_ROWS);
        const unsigned char* src = q + (size_t)tb * DQ_ROWS * n + c * 8;
        u32x2 v[DQ_ROWS];
#pragma unroll
        for (int r = 0; r < DQ_ROWS; ++r) v[r] = r < rows ? __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src + (size_t)r * n)) : u32x2{0u, 0u};
        const u32x2 s = *reinterpret_cast<const u32x2*>(scale + (size_t)(tb / (QBLOCK / DQ_ROWS)) * n + c * 8);
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(((s[e >> 2] >> (8 * (e & 3))) & 0xffu) << 23);
#pragma unroll
        for (int r = 0; r < DQ_ROWS; ++r) {
            u32x4 o;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[r][w], false);
                const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[r][w], true);
                const bf16x2 lo = {f2bf(a[0] * f[4 * w]), f2bf(a[1] * f[4 * w + 1])};
                const bf16x2 hi = {f2bf(b[0] * f[4 * w + 2]), f2bf(b[1] * f[4 * w + 3])};
                o[2 * w] = __builtin_bit_cast(uint32_t, lo);
                o[2 * w + 1] = __builtin_bit_cast(uint32_t, hi);
            }
            if (r < rows) __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(y + (size_t)(tb * DQ_ROWS + r) * ldy + c * 8));
        }
    }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// dw[m][n] = sum over tokens t of dy[t][m] x[t][n], x the checkpoint's values.  The tokens are cut into `splits` slices whose
// sums go to slabs [splits][M][N] and are added by a second kernel in a fixed order; one slice writes dw, or adds to it, itself.
struct DwParams {
    const bf16* dy;
    const unsigned char *q, *scale;
    float* out;                        // slabs, or dw when one slice covers all tokens
    int M, N, T, lddy, ldout;
    long long heads;                   // > 0: dy is head-major (features 64h .. 64h + 63 at dy + h * heads, rows of 64)
    int k_per_split;                   // a multiple of 64
    long long slab;                    // elements between the slabs
    int add;                           // out is dw and is added to
};

template <bool ADD>
__device__ __forceinline__ void put4(float* at, f32x4 v) {
    if (ADD) v += *reinterpret_cast<const f32x4*>(at);
    *reinterpret_cast<f32x4*>(at) = v;
}

struct DwItem {
    int m0, n0, split, kbeg, kend;
    __amdgpu_buffer_rsrc_t rA, rB, rS;
};

// Descriptors start at the slice's first token and end with its last one: tokens past the end read as zeros, and offsets
// stay small however many tokens there are.  A ragged tile reads its neighbours' columns; those outputs are not stored.
template <int BM, int BN>
__device__ __forceinline__ DwItem dw_item(const DwParams& p, int L, int ntm, int ntn) {
    DwItem it;
    const int tiles = ntm * ntn;
    it.split = L / tiles;
    const int t = L - it.split * tiles;
    int tm, tn;
    if (ntm >= ntn) { tm = t / ntn; tn = t - tm * ntn; } else { tn = t / ntm; tm = t - tn * ntm; }
    it.m0 = tm * BM;
    it.n0 = tn * BN;
    it.kbeg = it.split * p.k_per_split;
    it.kend = min(p.T, it.kbeg + p.k_per_split);
    const int k = it.kend - it.kbeg;
    const bf16* a = p.dy + (p.heads ? (size_t)(it.m0 >> 6) * p.heads : (size_t)it.m0) + (size_t)it.kbeg * p.lddy;
    const uint32_t ra = p.heads ? (uint32_t)(((size_t)(min(BM, (p.M - it.m0 + 63) & ~63) / 64 - 1) * p.heads + (size_t)k * 64) * 2)
                                : (uint32_t)(((size_t)(k - 1) * p.lddy + min(BM, p.M - it.m0)) * 2);
    it.rA = __builtin_amdgcn_make_buffer_rsrc((void*)a, 0, ra, 0x00020000);
    const int cols = min(BN, p.N - it.n0);
    it.rB = __builtin_amdgcn_make_buffer_rsrc((void*)(p.q + (size_t)it.kbeg * p.N + it.n0), 0, (uint32_t)((size_t)(k - 1) * p.N + cols), 0x00020000);
    it.rS = __builtin_amdgcn_make_buffer_rsrc((void*)(p.scale + (size_t)(it.kbeg / QBLOCK) * p.N + it.n0), 0,
                                              (uint32_t)((size_t)((k + QBLOCK - 1) / QBLOCK - 1) * p.N + cols), 0x00020000);
    return it;
}

// eight codes of one feature (eight tokens) to a bf16 fragment, exactly
__device__ __forceinline__ bf16x8 act8_fragment(u32x2 c, uint32_t code) {
    const float s = __uint_as_float(code << 23);
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], s, true);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], s, false), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], s, true);
    return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// 64x64 tile, eight waves, a ring of NS K steps (64 tokens) per workgroup, three workgroups to a compute unit.  Waves 0-3 hold
// 32x32 quarters of a step's first 32 tokens' product, waves 4-7 of the second's; their sums meet in LDS at the end.  Four
// waves with all 64 tokens took 9.2 us instead of 8.5 for 512 x 2048 from 1001 tokens, 12.2 instead of 10.9 for 2048 x 512 from
// 1500, but 4.4 instead of 4.9 from 33.
// LDS of one step: dy's image [64 tokens][64] bf16 (gemm_tiles.h), the codes' image [64 tokens][64] bytes whose 16-byte
// units u of token k sit at u ^ ((k >> 2) & 1) (the eight tokens that ds_read_b64_tr_b8 gathers then fall on different
// banks), and each quarter's 2 x 32 scale bytes.
constexpr int DW_A = 8192, DW_B = 4096, DW_STEP = DW_A + DW_B + 1024, DW_NS = 4, DW_PER = 2;
__global__ void __launch_bounds__(512) act8_dw_kernel(DwParams p, int ntm, int ntn, int total) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave >> 2, w = wave & 3;
    const int wm = w >> 1, wn = w & 1;
    const DwItem it = dw_item<64, 64>(p, xcd_remap(blockIdx.x, total), ntm, ntn);
    const uint32_t offA = stage_offset<true, 64>(wave * 64 + lane, p.lddy, p.heads);
    // waves 0-3 fetch the codes too, waves 4-7 the scales: lanes 0-7 the step's first 32 tokens' of a quarter's 32 features,
    // lanes 8-15 the second's; the others' offset lies outside every descriptor
    const int gk = (w * 64 + lane) >> 2, gc = ((w * 64 + lane) & 3) ^ ((gk >> 2) & 1);
    const uint32_t offB = (uint32_t)(gk * p.N + gc * 16);
    const uint32_t offS = lane < 16 ? (uint32_t)((lane >> 3) * p.N + wn * 32 + (lane & 7) * 4) : 0x80000000u;
    const uint32_t strideA = (uint32_t)p.lddy * 2u;
    const int nsteps = (it.kend - it.kbeg + BK - 1) / BK;
    auto stage = [&](int t, int buf) {
        char* l = smem + buf * DW_STEP;
        const uint32_t k = (uint32_t)t * BK;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(it.rA, LDS_PTR(l + wave * 1024), 16, offA, k * strideA, 0, 0);
        if (half == 0) __builtin_amdgcn_raw_ptr_buffer_load_lds(it.rB, LDS_PTR(l + DW_A + w * 1024), 16, offB, k * (uint32_t)p.N, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(it.rS, LDS_PTR(l + DW_A + DW_B + w * 256), 4, offS, (k / QBLOCK) * (uint32_t)p.N, 0, 0);
    };
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DW_NS - 1; ++s)
        if (s < nsteps) stage(s, s);
    int buf = 0, nbuf = DW_NS - 1;
    // addresses of this lane's fragment reads inside a step's images
    const int g = lane >> 4, i16 = lane & 15;
    uint32_t rdA[2], rdB[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = (wm * 32 + i * 16) >> 4, hk = ((i16 >> 2) | ((g & 1) << 2)) & 3;
        rdA[i] = (uint32_t)((half * 32 + 8 * g + (i16 >> 2)) * 128 + ((u ^ hk) << 5) + (i16 & 3) * 8);
        const int kb = 8 * g + (i16 >> 1);
        rdB[i] = (uint32_t)(DW_A + (half * 32 + kb) * 64 + (((wn * 2 + i) ^ ((kb >> 2) & 1)) << 4) + (i16 & 1) * 8);
    }
    const uint32_t rdS = (uint32_t)(DW_A + DW_B + w * 256 + half * 32 + i16);
    for (int t = 0; t < nsteps; ++t) {
        if (t + DW_NS - 2 < nsteps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DW_NS - 2) * DW_PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        PACED_PINNED_BARRIER();
        if (t + DW_NS - 1 < nsteps) stage(t + DW_NS - 1, nbuf);
        const uint32_t l = (uint32_t)(uintptr_t)LDS_PTR(smem + buf * DW_STEP);
        bf16x4 lo[2], hi[2];
        u32x2 c[2];
        uint32_t s[2];
        // (inline assembly: next to LDS-DMA the compiler would drain every load in flight ahead of a read it can see)
        asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                     "ds_read_b64_tr_b8 %4, %10\n\tds_read_b64_tr_b8 %5, %11\n\t"
                     "ds_read_u8 %6, %13\n\tds_read_u8 %7, %13 offset:16\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(c[0]), "=&v"(c[1]), "=&v"(s[0]), "=&v"(s[1])
                     : "v"(l + rdA[0]), "v"(l + rdA[1]), "v"(l + rdB[0]), "v"(l + rdB[1]), "n"(4 * 128), "v"(l + rdS)
                     : "memory");
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bf16x8 fb = act8_fragment(c[j], s[j]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, 0);
        }
        buf = buf + 1 == DW_NS ? 0 : buf + 1;
        nbuf = nbuf + 1 == DW_NS ? 0 : nbuf + 1;
    }
    __syncthreads();                                  // the last step has been read: its LDS takes the second half's sums
    f32x4* const sums = reinterpret_cast<f32x4*>(smem) + w * 256 + lane;
    if (half)
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[k * 64] = acc[k >> 1][k & 1];
    __syncthreads();
    if (half) return;
    float* out = p.out + (size_t)it.split * p.slab;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = it.m0 + wm * 32 + i * 16 + i16;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = it.n0 + wn * 32 + j * 16 + g * 4;
            const f32x4 v = acc[i][j] + sums[(i * 2 + j) * 64];
            if (m >= p.M || n >= p.N) continue;                                                      // N is a multiple of 16
            if (p.add) put4<true>(out + (size_t)m * p.ldout + n, v);
            else put4<false>(out + (size_t)m * p.ldout + n, v);
        }
    }
}

// 256x256 tiles: the phased kernel of gemm.hip (same ring order, phases, barriers and A halves) with B halves of codes: 8 KiB
// instead of 16, one LDS-DMA instruction per wave instead of two, half the fragment reads; a fragment is converted behind its
// phase's barrier.  Codes of a half: [64 tokens][128] bytes, 16-byte unit u of token k at u ^ (k & 7) ^ ((k >> 3) & 1) (the
// sixteen tokens that two lane groups gather lie on different banks); half h holds the h-th 32 features of every 64.  With each
// step's first B half every wave fetches the scales of its own 64 features.
// Instructions in flight behind a phase's wait (the six youngest half-tiles; B half 0 and its scales 2, A halves 2, B half 1 1):
// 11 after B half 0 and A half 0 were issued, 10 after B half 1 and A half 1.
// LDS: ring slots 0, 2, .. 8 are B halves (5 x 8 KiB), 1, 3, .. 9 A halves (5 x 16 KiB), three sets of scales (a set is read in
// its step and overwritten two steps on): 126 KiB.
constexpr int DP_B = 5 * 16384, DP_S = DP_B + 5 * 8192, DP_LDS = DP_S + 3 * 2048;

struct DwStep {
    __amdgpu_buffer_rsrc_t rA, rB, rS;
    uint32_t sA, sB, sS;
};
struct DwStream {
    DwItem it;
    int k, round;
    bool live;
    __device__ __forceinline__ DwStep take(const DwParams& p, int b, int G, int ntm, int ntn, int total, uint32_t strideA) {
        DwStep s;
        if (live) {
            s.rA = it.rA; s.rB = it.rB; s.rS = it.rS;
            s.sA = (uint32_t)k * strideA; s.sB = (uint32_t)k * (uint32_t)p.N; s.sS = (uint32_t)(k / QBLOCK) * (uint32_t)p.N;
            k += BK;
            if (it.kbeg + k >= it.kend) {
                const int L = item_of(b, ++round, G, total);
                if (L >= 0) { it = dw_item<256, 256>(p, L, ntm, ntn); k = 0; }
                else live = false;
            }
        } else {                       // past the last item: the same instructions through empty descriptors
            s.rA = __builtin_amdgcn_make_buffer_rsrc((void*)p.dy, 0, 0, 0x00020000);
            s.rB = __builtin_amdgcn_make_buffer_rsrc((void*)p.q, 0, 0, 0x00020000);
            s.rS = __builtin_amdgcn_make_buffer_rsrc((void*)p.scale, 0, 0, 0x00020000);
            s.sA = s.sB = s.sS = 0;
        }
        return s;
    }
};

__global__ void __launch_bounds__(512) act8_dw_phased_kernel(DwParams p, int ntm, int ntn, int total) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = w >> 2, wc = w & 3, g = lane >> 4, i16 = lane & 15;
    const int G = gridDim.x, b = blockIdx.x;

    uint32_t offA[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) offA[i] = stage_offset<true, 128>((i * 8 + w) * 64 + lane, p.lddy, p.heads);
    const int bk = (w * 64 + lane) >> 3, bc = ((w * 64 + lane) & 7) ^ (bk & 7) ^ ((bk >> 3) & 1);
    const uint32_t offB = (uint32_t)(bk * p.N + (bc >> 1) * 64 + (bc & 1) * 16);
    // lanes 0-15: the first 32 tokens' scales of the wave's 64 features, 16-31: the second's, the rest outside every descriptor
    const uint32_t offS = lane < 32 ? (uint32_t)((lane >> 4) * p.N + wc * 64 + (lane & 15) * 4) : 0x80000000u;
    const uint32_t strideA = (uint32_t)p.lddy * 2u;
    const uint32_t halfA = p.heads ? (uint32_t)(p.heads * 4) : 256u, halfB = 32u;
    char* const sw = smem + w * 1024;
    char* const ssc = smem + DP_S + w * 256;
#define DP_STAGE_A(st, slot, off) PACED_STAGE_HALF((st).rA, sw + ((slot) >> 1) * 16384, offA, (st).sA + (off))
#define DP_STAGE_B(st, slot, off) __builtin_amdgcn_raw_ptr_buffer_load_lds((st).rB, LDS_PTR(sw + DP_B + ((slot) >> 1) * 8192), 16, offB, (st).sB + (off), 0, 0)
#define DP_STAGE_S(st, set) __builtin_amdgcn_raw_ptr_buffer_load_lds((st).rS, LDS_PTR(ssc + (set) * 2048), 4, offS, (st).sS, 0, 0)

    const int L = item_of(b, 0, G, total);
    if (L < 0) return;
    DwStream st;
    st.it = dw_item<256, 256>(p, L, ntm, ntn);
    st.k = 0; st.round = 0; st.live = true;
    DwItem cur = st.it;
    {
        const DwStep c0 = st.take(p, b, G, ntm, ntn, total, strideA);
        const DwStep c1 = st.take(p, b, G, ntm, ntn, total, strideA);
        DP_STAGE_B(c0, 0, 0); DP_STAGE_S(c0, 0);
        DP_STAGE_A(c0, 1, 0);
        DP_STAGE_B(c0, 2, halfB);
        DP_STAGE_A(c0, 3, halfA);
        DP_STAGE_B(c1, 4, 0); DP_STAGE_S(c1, 1);
        DP_STAGE_A(c1, 5, 0);
        DP_STAGE_B(c1, 6, halfB);
        DP_STAGE_A(c1, 7, halfA);
    }
    asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (wr == 1) __builtin_amdgcn_s_barrier();       // second wave group runs one barrier behind
    DwStep c2 = st.take(p, b, G, ntm, ntn, total, strideA);

    f32x4 acc[8][4];
    bf16x8 fa[4][2], fb0[2][2], fb1[2][2];
    u32x2 cb[2][2];
    uint32_t sb[2][2];
    int base = 0, set = 0;                            // ring slot of this K step's first half-tile, its set of scales
    // fragment reads of one B half (inline assembly, waited for behind the phase's barrier like A's)
    auto read_b = [&](int slot, int half) {
        const uint32_t lb = (uint32_t)(uintptr_t)LDS_PTR(smem + DP_B + (slot >> 1) * 8192);
        const uint32_t ls = (uint32_t)(uintptr_t)LDS_PTR(ssc + set * 2048) + (uint32_t)(half * 32 + i16);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int k = 8 * g + (i16 >> 1);
            const uint32_t a = lb + (uint32_t)(k * 128 + (((wc * 2 + j) ^ (k & 7) ^ (g & 1)) << 4) + (i16 & 1) * 8);
            asm volatile("ds_read_b64_tr_b8 %0, %1" : "=v"(cb[j][0]) : "v"(a));
            asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(cb[j][1]) : "v"(a), "n"(32 * 128));
            if (j == 0) {
                asm volatile("ds_read_u8 %0, %1" : "=v"(sb[0][0]) : "v"(ls));
                asm volatile("ds_read_u8 %0, %1 offset:64" : "=v"(sb[0][1]) : "v"(ls));
            } else {
                asm volatile("ds_read_u8 %0, %1 offset:16" : "=v"(sb[1][0]) : "v"(ls));
                asm volatile("ds_read_u8 %0, %1 offset:80" : "=v"(sb[1][1]) : "v"(ls));
            }
        }
    };
    auto convert_b = [&](bf16x8 (&fb)[2][2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) fb[j][kk] = act8_fragment(cb[j][kk], sb[j][kk]);
    };
    for (int round = 0;;) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int nsteps = (cur.kend - cur.kbeg + BK - 1) / BK;
        for (int t = 0; t < nsteps; ++t) {
            const int sB0 = base, sA0 = ring_wrap(base + 1), sB1 = ring_wrap(base + 2), sA1 = ring_wrap(base + 3);
            const int d1 = ring_wrap(base + 8), d2 = ring_wrap(base + 9);      // phases 3 and 4 reuse sB0 and sA0
            const int next2 = set == 0 ? 2 : set - 1;                            // the set of step t + 2
            // ---- phase 1
            read_b(sB0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) fa[i][kk] = read_frag<true, 128, true>(smem + (sA0 >> 1) * 16384, wr * 64 + i * 16, kk, lane);
            DP_STAGE_B(c2, d1, 0);
            DP_STAGE_S(c2, next2);
            asm volatile("s_waitcnt vmcnt(11)" ::: "memory");
            PACED_PINNED_BARRIER();
            PACED_WAIT_LDS_READS();
            convert_b(fb0);
            quadrant_mfma<false>(fa, fb0, acc, 0, 0);
            PACED_PINNED_BARRIER();
            // ---- phase 2
            read_b(sB1, 1);
            DP_STAGE_A(c2, d2, 0);
            asm volatile("s_waitcnt vmcnt(11)" ::: "memory");
            PACED_PINNED_BARRIER();
            PACED_WAIT_LDS_READS();
            convert_b(fb1);
            quadrant_mfma<false>(fa, fb1, acc, 0, 1);
            PACED_PINNED_BARRIER();
            // ---- phase 3
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) fa[i][kk] = read_frag<true, 128, true>(smem + (sA1 >> 1) * 16384, wr * 64 + i * 16, kk, lane);
            DP_STAGE_B(c2, sB0, halfB);
            asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
            PACED_PINNED_BARRIER();
            PACED_WAIT_LDS_READS();
            quadrant_mfma<false>(fa, fb1, acc, 1, 1);
            PACED_PINNED_BARRIER();
            // ---- phase 4
            DP_STAGE_A(c2, sA0, halfA);
            c2 = st.take(p, b, G, ntm, ntn, total, strideA);
            base = ring_wrap(base + 4);
            set = set == 2 ? 0 : set + 1;
            asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
            PACED_PINNED_BARRIER();
            quadrant_mfma<false>(fa, fb0, acc, 1, 0);
            PACED_PINNED_BARRIER();
        }
        if (wr == 0) __builtin_amdgcn_s_barrier();       // both groups run their epilogues side by side (see gemm.hip)
        float* out = p.out + (size_t)cur.split * p.slab;
        auto store = [&](auto add) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int m = cur.m0 + CfgPhased::moff(wr, i) + i16;
                if (m >= p.M) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = cur.n0 + CfgPhased::noff(wc, j) + g * 4;
                    if (n < p.N) put4<add()>(out + (size_t)m * p.ldout + n, acc[i][j]);
                }
            }
        };
        if (p.add) store(std::true_type()); else store(std::false_type());
        const int Ln = item_of(b, ++round, G, total);
        if (Ln < 0) break;
        cur = dw_item<256, 256>(p, Ln, ntm, ntn);
        if (wr == 1) __builtin_amdgcn_s_barrier();       // fall one barrier behind again
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#undef DP_STAGE_A
#undef DP_STAGE_B
#undef DP_STAGE_S
}

// dw (+)= the slabs' sum, slab by slab
__global__ void __launch_bounds__(256) slab_sum_kernel(const float* __restrict__ slabs, int count, long long slab, float* dw, int lddw,
                                                       int M, int N, int accumulate) {
    const int n4 = N >> 2;
    const long long total = (long long)M * n4;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < total; id += (long long)gridDim.x * 256) {
        const int m = (int)(id / n4), c = (int)(id - (long long)m * n4);
        const float* src = slabs + (size_t)m * N + c * 4;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < count; ++k) s += *reinterpret_cast<const f32x4*>(src + (size_t)k * slab);
        float* dst = dw + (size_t)m * lddw + c * 4;
        if (accumulate) s += *reinterpret_cast<const f32x4*>(dst);
        *reinterpret_cast<f32x4*>(dst) = s;
    }
}

// Which tiles, and how many slices of the tokens: the plan with the least time by what the kernels were measured to take.  A
// 64x64 tile's workgroup 3.2 us and 0.31 for each K step of 64 tokens, half of that more for each further workgroup of its
// compute unit; a 256x256 tile's 10 us and 1.4 for a step; several slices 3 us for the second kernel, and their slabs written
// and read at 4.5 and 7.5 TB/s.  Good to about a tenth.  Both sides of it, in us: 1001 tokens, 768 x 768, 64x64 tiles, 1 slice
// 8.0, 4 slices 14.0; 4352, 512 x 512, 4 slices 12.7, 1 slice 23.1, 12 slices 16.6; 4352, 2304 x 768, 64x64 30.5, 256x256 38.5;
// 8704, 768 x 768, 5 slices 25.5, 4 slices 27.7; 8704, 2304 x 768, 64x64 56, 256x256 50; 139264, 768 x 768, 64x64 300, 256x256 156.
struct DwPlan { int tile, ntm, ntn, splits, k_per_split; };
DwPlan dw_plan(int T, int M, int N) {
    const int ktiles = (T + BK - 1) / BK, cus = paced_cu_count();
    const double slab = (double)M * N * 8.;
    DwPlan pl = {};
    double best = 1e300;
    for (int tile = 64; tile <= 256; tile += 192) {
        const long long tiles = (long long)((M + tile - 1) / tile) * ((N + tile - 1) / tile);
        for (const int c : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 0, -1}) {                     // 0, -1: one or three tiles to a compute unit
            int splits = c > 0 ? c : (int)((c ? 3 : 1) * cus / tiles < 64 ? (c ? 3 : 1) * cus / tiles : 64);
            if (splits > ktiles || splits < 1) continue;
            const int per = (ktiles + splits - 1) / splits;
            splits = (ktiles + per - 1) / per;
            const double groups = (double)((tiles * splits + cus - 1) / cus);
            double us = tile == 64 ? 3.2 + per * 0.31 * (0.5 + 0.5 * groups) : 10. + per * 1.4 * groups;
            if (splits > 1) us += 3. + splits * slab / (tile == 64 ? 4.5e6 : 7.5e6);
            if (us < best) { best = us; pl = DwPlan{tile, (M + tile - 1) / tile, (N + tile - 1) / tile, splits, per * BK}; }
        }
    }
    return pl;
}

thread_local int t_last_tile = 0;      // tile edge of this thread's most recent weight gradient

int flat_blocks(long long items) {
    const long long g = (items + 255) / 256;
    return (int)(g < 1 ? 1 : g > 16384 ? 16384 : g);
}

}  // namespace

extern "C" int paced_act8_quantize(const void* x, int ldx, void* q, void* scale, int T, int n, void* stream) {
    PACED_CHECK_ARG(T >= 0 && T <= MAX_T && n > 0 && n % 16 == 0, "paced_act8_quantize: need T >= 0, at most %d, and n a multiple of 16 (T=%d n=%d)", MAX_T, T, n);
    if (T == 0) return PACED_OK;
    PACED_CHECK_ARG(x && q && scale, "paced_act8_quantize: null operand");
    PACED_CHECK_ARG(ldx >= n && ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)q | (uintptr_t)scale) & 15) == 0,
                    "paced_act8_quantize: 16-byte aligned operands and a row stride of at least n and a multiple of 8 are needed (ldx=%d)", ldx);
    const int nblk = (T + QBLOCK - 1) / QBLOCK;
    hipLaunchKernelGGL(act8_quantize_kernel, dim3(flat_blocks((long long)nblk * (n >> 1))), dim3(256), 0, (hipStream_t)stream,
                       (const bf16*)x, ldx, (unsigned char*)q, (unsigned char*)scale, T, n, nblk);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}

extern "C" int paced_act8_dequantize(const void* q, const void* scale, void* y, int ldy, int T, int n, void* stream) {
    PACED_CHECK_ARG(T >= 0 && T <= MAX_T && n > 0 && n % 16 == 0, "paced_act8_dequantize: need T >= 0, at most %d, and n a multiple of 16 (T=%d n=%d)", MAX_T, T, n);
    if (T == 0) return PACED_OK;
    PACED_CHECK_ARG(q && scale && y, "paced_act8_dequantize: null operand");
    PACED_CHECK_ARG(ldy >= n && ldy % 8 == 0 && (((uintptr_t)y | (uintptr_t)q | (uintptr_t)scale) & 15) == 0,
                    "paced_act8_dequantize: 16-byte aligned operands and a row stride of at least n and a multiple of 8 are needed (ldy=%d)", ldy);
    hipLaunchKernelGGL(act8_dequantize_kernel, dim3(flat_blocks((long long)((T + DQ_ROWS - 1) / DQ_ROWS) * (n >> 3))), dim3(256), 0, (hipStream_t)stream,
                       (const unsigned char*)q, (const unsigned char*)scale, (bf16*)y, ldy, T, n);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}

extern "C" int paced_act8_last_tile(void) { return t_last_tile; }

extern "C" size_t paced_act8_dweight_workspace_bytes(int T, int M, int N) {
    if (T <= 0 || T > MAX_T || M <= 0 || N <= 0) return 0;
    const DwPlan pl = dw_plan(T, M, N);
    return pl.splits == 1 ? 0 : (size_t)pl.splits * M * N * 4;
}

extern "C" int paced_act8_dweight(const void* dy, int lddy, long long dy_heads, const void* q, const void* scale, float* dw, int lddw,
                                  int T, int M, int N, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    PACED_CHECK_ARG(T >= 0 && T <= MAX_T && M > 0 && N > 0 && M % 8 == 0 && N % 16 == 0,
                    "paced_act8_dweight: need T >= 0, at most %d, M a multiple of 8 and N a multiple of 16 (T=%d M=%d N=%d)", MAX_T, T, M, N);
    PACED_CHECK_ARG(dw && lddw >= N && lddw % 4 == 0 && ((uintptr_t)dw & 15) == 0,
                    "paced_act8_dweight: dw must be 16-byte aligned with a row stride of at least N and a multiple of 4 (lddw=%d)", lddw);
    PACED_CHECK_ARG(T == 0 || (dy && q && scale && (((uintptr_t)dy | (uintptr_t)q | (uintptr_t)scale) & 15) == 0), "paced_act8_dweight: dy, q and scale must be 16-byte aligned");
    if (dy_heads > 0) PACED_CHECK_ARG(lddy == 64 && M % 64 == 0 && dy_heads >= (long long)T * 64 && dy_heads % 8 == 0,
                                      "paced_act8_dweight: a head-major dy has rows of 64, M a multiple of 64 and heads at least T * 64 elements apart");
    else PACED_CHECK_ARG(T == 0 || (lddy >= M && lddy % 8 == 0), "paced_act8_dweight: dy's row stride must be at least M and a multiple of 8 (lddy=%d)", lddy);
    hipStream_t s = (hipStream_t)stream;
    if (T == 0) {                                   // an empty sum
        if (accumulate) return PACED_OK;
        hipLaunchKernelGGL(slab_sum_kernel, dim3(flat_blocks((long long)M * (N >> 2))), dim3(256), 0, s, nullptr, 0, 0LL, dw, lddw, M, N, 0);
        PACED_CHECK_LAUNCH();
        return PACED_OK;
    }
    const DwPlan pl = dw_plan(T, M, N);
    const size_t need = pl.splits == 1 ? 0 : (size_t)pl.splits * M * N * 4;
    PACED_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                    "paced_act8_dweight: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need, workspace_bytes);
    // Offsets inside one slice are 32-bit: `reach` tokens of dy (a tile's four heads, or whole rows) and of the codes span less than
    // 2 GiB.  Where the plan's slices are longer, the tokens go by in passes of at most as many slices, each added to the one
    // before (139264 tokens, 8192 x 2048: two).
    const long long most = (1ll << 31) - 1, apart = dy_heads > 0 ? 8 * dy_heads : 0;
    const long long by_dy = (most - apart) / (dy_heads > 0 ? 128 : 2ll * lddy + 128), by_codes = most / N;
    const long long reach = (by_dy < by_codes ? by_dy : by_codes) / BK * BK;
    PACED_CHECK_ARG(apart < most && reach > 0, "paced_act8_dweight: 64 tokens of dy (lddy=%d, heads %lld elements apart) span more than 2 GiB", lddy, dy_heads);
    const int passes = (int)((T + pl.splits * reach - 1) / (pl.splits * reach));
    if (pl.tile == 256) {
        static PerDeviceOnce once;
        bool& attr_set = once.flag();
        if (!attr_set) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&act8_dw_phased_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, DP_LDS);
            if (e != hipSuccess) { paced_set_error("paced_act8_dweight: hipFuncSetAttribute(%d bytes LDS) failed: %s", DP_LDS, hipGetErrorString(e)); return PACED_ERR_HIP; }
            attr_set = true;
        }
    }
    t_last_tile = pl.tile;
    const int ktiles = (T + BK - 1) / BK, a_pass = (ktiles + passes - 1) / passes;
    for (int first = 0; first < ktiles; first += a_pass) {
        const int steps = a_pass < ktiles - first ? a_pass : ktiles - first, t0 = first * BK;
        const int per = (steps + pl.splits - 1) / pl.splits, splits = (steps + per - 1) / per;
        const int add = accumulate || first > 0;
        DwParams p;
        p.dy = (const bf16*)dy + (size_t)t0 * lddy;                  // (rows of 64 where it is head-major)
        p.q = (const unsigned char*)q + (size_t)t0 * N;
        p.scale = (const unsigned char*)scale + (size_t)(t0 / QBLOCK) * N;
        p.M = M; p.N = N; p.T = first + steps < ktiles ? steps * BK : T - t0; p.lddy = lddy; p.heads = dy_heads > 0 ? dy_heads : 0;
        p.k_per_split = per * BK;
        p.out = need ? (float*)workspace : dw;
        p.ldout = need ? N : lddw;
        p.slab = (long long)M * N;
        p.add = !need && add;
        const int total = pl.ntm * pl.ntn * splits, cus = paced_cu_count();
        if (pl.tile == 256) hipLaunchKernelGGL(act8_dw_phased_kernel, dim3(total < cus ? total : cus), dim3(512), DP_LDS, s, p, pl.ntm, pl.ntn, total);
        else hipLaunchKernelGGL(act8_dw_kernel, dim3(total), dim3(512), DW_NS * DW_STEP, s, p, pl.ntm, pl.ntn, total);
        PACED_CHECK_LAUNCH();
        if (need) {
            hipLaunchKernelGGL(slab_sum_kernel, dim3(flat_blocks((long long)M * (N >> 2))), dim3(256), 0, s, p.out, splits, p.slab, dw, lddw, M, N, add);
            PACED_CHECK_LAUNCH();
        }
    }
    return PACED_OK;
}
