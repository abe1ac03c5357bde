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
#include "gemm_tiles.h"

namespace {

constexpr int QBLOCK = 32;                 // tokens per scale
constexpr int MIN_CODE = 127 - 117, MAX_CODE = 127 + 120, NAN_CODE = 255;

// ------------------------------------------------------------------------------------------------ writing and reading
// One thread per 32 tokens x 8 features: 32 loads of 16 bytes in flight, the maxima in its own registers (integer maxima of
// the magnitudes' bits, two features to a register), no exchange between lanes.
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
__global__ void __launch_bounds__(256) act8_quantize_kernel(const bf16* __restrict__ x, int ldx, unsigned char* __restrict__ q,
                                                            unsigned char* __restrict__ scale, int T, int n, int nblk) {
    const int chunks = n >> 3;
    const long long total = (long long)nblk * chunks;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < total; id += (long long)gridDim.x * 256) {
        const int blk = (int)(id / chunks), c = (int)(id - (long long)blk * chunks);
        const int rows = min(QBLOCK, T - blk * QBLOCK);
        const bf16* src = x + (size_t)blk * QBLOCK * ldx + c * 8;
        u32x4 v[QBLOCK];
#pragma unroll
        for (int r = 0; r < QBLOCK; ++r) v[r] = r < rows ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + (size_t)r * ldx)) : u32x4{0u, 0u, 0u, 0u};
        u16x2 top[4] = {};
#pragma unroll
        for (int r = 0; r < QBLOCK; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) top[j] = __builtin_elementwise_max(top[j], __builtin_bit_cast(u16x2, v[r][j] & 0x7fff7fffu));
        float inv[8], lim[8];
        uint32_t bad = 0;                  // bit e: feature e of this thread holds a value that is not finite
        uint32_t code[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int bits = top[e >> 1][e & 1];
            int k = (bits >> 7) - 8 + ((bits & 0x7f) > 0x60 ? 1 : 0);        // 448 = 1.75 * 2^8
            k = max(k, MIN_CODE);
            inv[e] = __uint_as_float((uint32_t)(254 - k) << 23);
            lim[e] = k == MAX_CODE ? 240.f : 448.f;
            if (bits >= 0x7f80) { bad |= 1u << e; k = NAN_CODE; }
            code[e >> 2] |= (uint32_t)k << (8 * (e & 3));
        }
        *reinterpret_cast<u32x2*>(scale + (size_t)blk * n + c * 8) = u32x2{code[0], code[1]};
        unsigned char* dst = q + (size_t)blk * QBLOCK * n + c * 8;
#pragma unroll
        for (int r = 0; r < QBLOCK; ++r) {
            u32x2 o;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t u = v[r][h * 2 + (e >> 1)];
                    const float y = __uint_as_float((e & 1) ? (u & 0xffff0000u) : (u << 16)) * inv[h * 4 + e];
                    f[e] = fminf(fmaxf(y, -lim[h * 4 + e]), lim[h * 4 + e]);
                }
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                w = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
                o[h] = (uint32_t)w;
            }
            if (bad) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((bad >> e) & 1u) o[e >> 2] |= 0x7fu << (8 * (e & 3));
            }
            if (r < rows) __builtin_nontemporal_store(o, reinterpret_cast<u32x2*>(dst + (size_t)r * n));
        }
    }
}

// One thread per 8 tokens x 16 features.
__global__ void __launch_bounds__(256) act8_dequantize_kernel(const unsigned char* __restrict__ q, const unsigned char* __restrict__ scale,
                                                              bf16* __restrict__ y, int ldy, int T, int n) {
    const int chunks = n >> 4;
    const long long total = (long long)((T + 7) >> 3) * chunks;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < total; id += (long long)gridDim.x * 256) {
        const int t8 = (int)(id / chunks), c = (int)(id - (long long)t8 * chunks);
        const int rows = min(8, T - t8 * 8);
        u32x4 v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = r < rows ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(q + (size_t)(t8 * 8 + r) * n + c * 16)) : u32x4{0u, 0u, 0u, 0u};
        const u32x4 s = *reinterpret_cast<const u32x4*>(scale + (size_t)(t8 >> 2) * n + c * 16);
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(((s[e >> 2] >> (8 * (e & 3))) & 0xffu) << 23);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            u32x4 o[2];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[r][w], false);
                const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v[r][w], true);
                const bf16x2 lo = {f2bf(a[0] * f[4 * w]), f2bf(a[1] * f[4 * w + 1])};
                const bf16x2 hi = {f2bf(b[0] * f[4 * w + 2]), f2bf(b[1] * f[4 * w + 3])};
                o[w >> 1][(w & 1) * 2] = __builtin_bit_cast(uint32_t, lo);
                o[w >> 1][(w & 1) * 2 + 1] = __builtin_bit_cast(uint32_t, hi);
            }
            if (r < rows) {
                bf16* dst = y + (size_t)(t8 * 8 + r) * ldy + c * 16;
                __builtin_nontemporal_store(o[0], reinterpret_cast<u32x4*>(dst));
                __builtin_nontemporal_store(o[1], reinterpret_cast<u32x4*>(dst + 8));
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// dw[m][n] = sum over tokens t of dy[t][m] x[t][n], x the checkpoint's values.  The tokens are cut into `splits` slices whose
// sums go to slabs [splits][M][N] and are added by a second kernel in a fixed order; one slice writes dw itself.
struct DwParams {
    const bf16* dy;
    const unsigned char *q, *scale;
    float* out;                        // slabs, or dw when one slice covers all tokens
    int M, N, T, lddy, ldout;
    long long heads;                   // > 0: dy is head-major (features 64h .. 64h + 63 at dy + h * heads, rows of 64)
    int k_per_split;                   // a multiple of 64
    long long slab;                    // elements between the slabs
};

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

// 64x64 tile, four waves of 32x32, a ring of NS K steps (64 tokens) per workgroup, three workgroups to a compute unit.
// LDS of one step: dy's image [64 tokens][64] bf16 (gemm_tiles.h), the codes' image [64 tokens][64] bytes whose 16-byte
// units u of token k sit at u ^ ((k >> 2) & 1) (the eight tokens that ds_read_b64_tr_b8 gathers then fall on different
// banks), and each wave's 2 x 32 scale bytes.
constexpr int DW_A = 8192, DW_B = 4096, DW_STEP = DW_A + DW_B + 1024, DW_NS = 4, DW_PER = 4;
__global__ void __launch_bounds__(256) act8_dw_kernel(DwParams p, int ntm, int ntn, int total) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = w >> 1, wn = w & 1;
    const DwItem it = dw_item<64, 64>(p, xcd_remap(blockIdx.x, total), ntm, ntn);
    uint32_t offA[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) offA[i] = stage_offset<true, 64>((i * 4 + w) * 64 + lane, p.lddy, p.heads);
    const int gk = (w * 64 + lane) >> 2, gc = ((w * 64 + lane) & 3) ^ ((gk >> 2) & 1);
    const uint32_t offB = (uint32_t)(gk * p.N + gc * 16);
    // lanes 0-7: the step's first 32 tokens' scales of this wave's 32 features, lanes 8-15: the second's; the others' offset
    // lies outside every descriptor
    const uint32_t offS = lane < 16 ? (uint32_t)((lane >> 3) * p.N + wn * 32 + (lane & 7) * 4) : 0x80000000u;
    const uint32_t strideA = (uint32_t)p.lddy * 2u;
    const int nsteps = (it.kend - it.kbeg + BK - 1) / BK;
    auto stage = [&](int t, int buf) {
        char* l = smem + buf * DW_STEP;
        const uint32_t k = (uint32_t)t * BK;
#pragma unroll
        for (int i = 0; i < 2; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(it.rA, LDS_PTR(l + (i * 4 + w) * 1024), 16, offA[i], k * strideA, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(it.rB, LDS_PTR(l + DW_A + w * 1024), 16, offB, k * (uint32_t)p.N, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(it.rS, LDS_PTR(l + DW_A + DW_B + w * 256), 4, offS, (k / QBLOCK) * (uint32_t)p.N, 0, 0);
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
    // addresses of this lane's fragment reads inside a step's images (kk = 0; kk = 1 is 32 tokens on)
    const int g = lane >> 4, i16 = lane & 15;
    uint32_t rdA[2], rdB[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = (wm * 32 + i * 16) >> 4, hk = ((i16 >> 2) | ((g & 1) << 2)) & 3;
        rdA[i] = (uint32_t)((8 * g + (i16 >> 2)) * 128 + ((u ^ hk) << 5) + (i16 & 3) * 8);
        const int kb = 8 * g + (i16 >> 1);
        rdB[i] = (uint32_t)(DW_A + kb * 64 + (((wn * 2 + i) ^ ((kb >> 2) & 1)) << 4) + (i16 & 1) * 8);
    }
    const uint32_t rdS = (uint32_t)(DW_A + DW_B + w * 256 + i16);
    for (int t = 0; t < nsteps; ++t) {
        if (t + DW_NS - 2 < nsteps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DW_NS - 2) * DW_PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        PACED_PINNED_BARRIER();
        if (t + DW_NS - 1 < nsteps) stage(t + DW_NS - 1, nbuf);
        const uint32_t l = (uint32_t)(uintptr_t)LDS_PTR(smem + buf * DW_STEP);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x4 lo[2], hi[2];
            u32x2 c[2];
            uint32_t s[2];
            // (inline assembly: next to LDS-DMA the compiler would drain every load in flight ahead of a read it can see)
            asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                         "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                         "ds_read_b64_tr_b8 %4, %10 offset:%14\n\tds_read_b64_tr_b8 %5, %11 offset:%14\n\t"
                         "ds_read_u8 %6, %15 offset:%16\n\tds_read_u8 %7, %15 offset:%17\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(c[0]), "=&v"(c[1]), "=&v"(s[0]), "=&v"(s[1])
                         : "v"(l + rdA[0]), "v"(l + rdA[1]), "v"(l + rdB[0]), "v"(l + rdB[1]), "n"(kk * 32 * 128), "n"(kk * 32 * 128 + 4 * 128),
                           "n"(kk * 32 * 64), "v"(l + rdS), "n"(kk * 32), "n"(kk * 32 + 16)
                         : "memory");
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bf16x8 fb = act8_fragment(c[j], s[j]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, 0);
            }
        }
        buf = buf + 1 == DW_NS ? 0 : buf + 1;
        nbuf = nbuf + 1 == DW_NS ? 0 : nbuf + 1;
    }
    float* out = p.out + (size_t)it.split * p.slab;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = it.m0 + wm * 32 + i * 16 + i16;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = it.n0 + wn * 32 + j * 16 + g * 4;
            if (n < p.N) *reinterpret_cast<f32x4*>(out + (size_t)m * p.ldout + n) = acc[i][j];        // N is a multiple of 16
        }
    }
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

struct DwPlan { int ntm, ntn, splits, k_per_split; };
DwPlan dw_plan(int T, int M, int N) {
    DwPlan pl;
    pl.ntm = (M + 63) / 64;
    pl.ntn = (N + 63) / 64;
    const int ktiles = (T + BK - 1) / BK;
    const long long tiles = (long long)pl.ntm * pl.ntn, slots = 3LL * paced_cu_count();
    long long splits = tiles >= slots ? 1 : slots / tiles;
    if (splits > (ktiles + 3) / 4) splits = (ktiles + 3) / 4;
    const int per = (int)((ktiles + splits - 1) / splits);
    pl.k_per_split = per * BK;
    pl.splits = (ktiles + per - 1) / per;
    return pl;
}

int flat_blocks(long long items) {
    const long long g = (items + 255) / 256;
    return (int)(g < 1 ? 1 : g > 16384 ? 16384 : g);
}

}  // namespace

extern "C" int paced_act8_quantize(const void* x, int ldx, void* q, void* scale, int T, int n, void* stream) {
    PACED_CHECK_ARG(T >= 0 && n > 0 && n % 16 == 0, "paced_act8_quantize: need T >= 0 and n a multiple of 16 (T=%d n=%d)", T, n);
    if (T == 0) return PACED_OK;
    PACED_CHECK_ARG(x && q && scale, "paced_act8_quantize: null operand");
    PACED_CHECK_ARG(ldx >= n && ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)q | (uintptr_t)scale) & 15) == 0,
                    "paced_act8_quantize: 16-byte aligned operands and a row stride of at least n and a multiple of 8 are needed (ldx=%d)", ldx);
    const int nblk = (T + QBLOCK - 1) / QBLOCK;
    hipLaunchKernelGGL(act8_quantize_kernel, dim3(flat_blocks((long long)nblk * (n >> 3))), dim3(256), 0, (hipStream_t)stream,
                       (const bf16*)x, ldx, (unsigned char*)q, (unsigned char*)scale, T, n, nblk);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}

extern "C" int paced_act8_dequantize(const void* q, const void* scale, void* y, int ldy, int T, int n, void* stream) {
    PACED_CHECK_ARG(T >= 0 && n > 0 && n % 16 == 0, "paced_act8_dequantize: need T >= 0 and n a multiple of 16 (T=%d n=%d)", T, n);
    if (T == 0) return PACED_OK;
    PACED_CHECK_ARG(q && scale && y, "paced_act8_dequantize: null operand");
    PACED_CHECK_ARG(ldy >= n && ldy % 8 == 0 && (((uintptr_t)y | (uintptr_t)q | (uintptr_t)scale) & 15) == 0,
                    "paced_act8_dequantize: 16-byte aligned operands and a row stride of at least n and a multiple of 8 are needed (ldy=%d)", ldy);
    hipLaunchKernelGGL(act8_dequantize_kernel, dim3(flat_blocks((long long)((T + 7) / 8) * (n >> 4))), dim3(256), 0, (hipStream_t)stream,
                       (const unsigned char*)q, (const unsigned char*)scale, (bf16*)y, ldy, T, n);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}

extern "C" size_t paced_act8_dweight_workspace_bytes(int T, int M, int N, int accumulate) {
    if (T <= 0 || M <= 0 || N <= 0) return 0;
    const DwPlan pl = dw_plan(T, M, N);
    return pl.splits == 1 && !accumulate ? 0 : (size_t)pl.splits * M * N * 4;
}

extern "C" int paced_act8_dweight(const void* dy, int lddy, long long dy_heads, const void* q, const void* scale, float* dw, int lddw,
                                  int T, int M, int N, int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    PACED_CHECK_ARG(T >= 0 && M > 0 && N > 0 && M % 8 == 0 && N % 16 == 0,
                    "paced_act8_dweight: need T >= 0, M a multiple of 8 and N a multiple of 16 (T=%d M=%d N=%d)", T, M, N);
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
    const size_t need = paced_act8_dweight_workspace_bytes(T, M, N, accumulate);
    PACED_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                    "paced_act8_dweight: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need, workspace_bytes);
    // offsets inside one slice are 32-bit
    const unsigned long long span = (dy_heads > 0 ? 4ull * dy_heads : (unsigned long long)pl.k_per_split * lddy) * 2 + (unsigned long long)pl.k_per_split * 128;
    PACED_CHECK_ARG(span < (1ull << 31) && (unsigned long long)pl.k_per_split * N < (1ull << 31),
                    "paced_act8_dweight: a slice of %d tokens spans more than 2 GiB; pass fewer tokens at a time", pl.k_per_split);
    DwParams p;
    p.dy = (const bf16*)dy; p.q = (const unsigned char*)q; p.scale = (const unsigned char*)scale;
    p.M = M; p.N = N; p.T = T; p.lddy = lddy; p.heads = dy_heads > 0 ? dy_heads : 0;
    p.k_per_split = pl.k_per_split;
    p.out = need ? (float*)workspace : dw;
    p.ldout = need ? N : lddw;
    p.slab = (long long)M * N;
    const int total = pl.ntm * pl.ntn * pl.splits;
    hipLaunchKernelGGL(act8_dw_kernel, dim3(total), dim3(256), DW_NS * DW_STEP, s, p, pl.ntm, pl.ntn, total);
    PACED_CHECK_LAUNCH();
    if (need) {
        hipLaunchKernelGGL(slab_sum_kernel, dim3(flat_blocks((long long)M * (N >> 2))), dim3(256), 0, s, p.out, pl.splits, p.slab, dw, lddw, M, N, accumulate);
        PACED_CHECK_LAUNCH();
    }
    return PACED_OK;
}
