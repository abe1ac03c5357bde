// Softmax cross entropy of a linear head over a large vocabulary, without its logits:
//   z = scale h w^T      lse_r = log sum_v exp z_rv      loss_r = lse_r - z_r,label (0 for an ignored row)
//   P_rv = g_r (exp(z_rv - lse_r) - [v = label_r])       dh = scale P w      dw = scale P^T h
// Forward: one product whose epilogue (EPI_CE_STATS in gemm.hip) leaves a maximum and a sum for every row and 64 columns, and
// a second kernel that joins them; the logits never leave the registers.  The label's term is kept out of the sums, so that
// a confident row's loss log(1 + sum of the others / its own) keeps its relative precision.  So does its gradient where the
// backward pass is given the losses: the label's entry is then g (exp(-loss) - 1).
// Backward: the vocabulary goes by in pieces.  A piece's logits are computed again and leave as P in bf16 (the MFMA operand
// type; half a step of 2^-8 relative to each entry, as paced_cross_entropy's dlogits), which feeds the two other products.  What
// the label's entry, the largest of a row, loses in that rounding is given back where dh is finished.  dw takes P's low part too
// up to 64 rows, where it costs little (ce_dw_few_kernel; 32128 x 768, backward pass of 64 rows 47.7 us, of 65 46.6); beyond, a
// second product of 2 R V d operations would be the price, and dw is off by up to 2^-8 of each addend, whether one row or many
// make up an element: measured 0.0017 of its norm before its own rounding (0.0024 with it, where a result that is only rounded at
// the end has 0.0017).
// dh is summed over pieces and slices of a piece in fp32 slabs with one owner per element, dw is complete with its piece:
// nothing is added atomically, equal inputs give equal bits.
// Matrix-core bound: 2 R V d operations forward, three times that backward.  Measured, loss and both gradients: 8192 rows x
// 50001 entries x 1024 in 2.9 to 3.0 ms (1.14 PFLOP/s over the four products), 1088 x 32128 x 768 in 254
// to 280 us on different cards (0.77 to 0.85 PFLOP/s: 4.25 x 125.5 tiles of 256 do not fill whole rounds of 256 compute units), 36
// more where dw is added to in fp32 (148 MB more, 27 us of them);
// the loss of 16 rows 15 us, of which the weights' 49 MB take 11.
#include "gemm.h"
#include "gemm_tiles.h"
#include <cmath>

namespace {

constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float mx = fmaxf(m, m2), at = mx == -INFINITY ? 0.f : mx;
    s = s * __builtin_amdgcn_exp2f(m - at) + s2 * __builtin_amdgcn_exp2f(m2 - at);
    m = mx;
}

// RPB rows of a workgroup, 256 / RPB threads over the column groups of each: 8 (64-byte runs of a group's row statistics), or
// 1 where there are too few rows to fill the chip
template <int RPB>
__global__ void __launch_bounds__(256) ce_join_kernel(const f32x2* __restrict__ part, int groups, const float* __restrict__ target,
                                                      const long long* __restrict__ labels, long long ignore, int V,
                                                      float* __restrict__ loss, float* __restrict__ lse, int R) {
    constexpr int K = 256 / RPB, AHEAD = RPB == 1 ? 4 : 8;
    __shared__ f32x2 sh[4][RPB];
    const int r = threadIdx.x % RPB, k = threadIdx.x / RPB;
    const int row = blockIdx.x * RPB + r, rr = min(row, R - 1);
    const long long label = labels[rr];
    const float t = target[rr];
    float m = -INFINITY, s = 0.f;
    int g = k;
    for (; g + (AHEAD - 1) * K < groups; g += AHEAD * K) {        // that many loads in flight
        f32x2 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = part[(size_t)(g + i * K) * R + rr];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) join(m, s, v[i][0], v[i][1]);
    }
    for (; g < groups; g += K) {
        const f32x2 v = part[(size_t)g * R + rr];
        join(m, s, v[0], v[1]);
    }
#pragma unroll
    for (int o = RPB; o < 64; o <<= 1) join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
    if ((threadIdx.x & 63) < RPB) sh[threadIdx.x >> 6][r] = f32x2{m, s};
    __syncthreads();
    if (threadIdx.x >= RPB || row >= R) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) join(m, s, sh[w][r][0], sh[w][r][1]);
    if (label == ignore || label < 0 || label >= V) {
        loss[row] = 0.f;
        if (lse) lse[row] = m * LN2 + logf(s);
        return;
    }
    const float t2 = t * LOG2E;                                 // (written for a label that counts; garbage otherwise)
    float l;
    if (m == -INFINITY) l = s == 0.f ? 0.f : s;                 // no other entry (or a NaN among them)
    else if (t2 >= m) l = log1pf(s * __builtin_amdgcn_exp2f(m - t2));
    else l = (m - t2) * LN2 + logf(s + __builtin_amdgcn_exp2f(t2 - m));
    loss[row] = l;
    if (lse) lse[row] = t + l;
}

// dh = bf16 of the slabs' sum and of scale err[r] w[label], the label's entry's share that P's rounding lost (labels NULL: the
// sum alone).  G groups of a workgroup's threads add every G-th slab each, group by group in the end: 8 where one thread to
// eight features leaves compute units without work (128 rows x 768 from 42 slabs:
// one group 15 us, eight 5), else 1.
template <int G>
__global__ void __launch_bounds__(256) ce_dh_kernel(const float* __restrict__ slabs, int count, long long slab, bf16* __restrict__ dh, int lddh, int R, int d,
                                                    const long long* __restrict__ labels, long long ignore, int V, const float* __restrict__ err,
                                                    const bf16* __restrict__ w, int ldw, float scale) {
    constexpr int L = 256 / G;
    __shared__ f32x4 sh[G > 1 ? 2 * 256 : 1];
    const int d8 = d >> 3, group = threadIdx.x / L, l = threadIdx.x % L;
    const long long total = (long long)R * d8;
    for (long long id0 = (long long)blockIdx.x * L; id0 < total; id0 += (long long)gridDim.x * L) {
        const long long id = id0 + l < total ? id0 + l : total - 1;
        const bool ok = id0 + l < total && group == 0;
        const int r = (int)(id / d8), c = (int)(id - (long long)r * d8);
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        bf16x8 x = {};
        float e = 0.f;
        if (ok && labels) {                                  // requested ahead of the slabs, added after them
            const long long label = labels[r];
            if (label != ignore && label >= 0 && label < V) {
                x = *reinterpret_cast<const bf16x8*>(w + (size_t)label * ldw + c * 8);
                e = scale * err[r];
            }
        }
        for (int k = group; k < count; k += G) {
            const float* src = slabs + (size_t)k * slab + (size_t)r * d + c * 8;
            a += *reinterpret_cast<const f32x4*>(src);
            b += *reinterpret_cast<const f32x4*>(src + 4);
        }
        if (G > 1) {
            sh[threadIdx.x] = a;
            sh[256 + threadIdx.x] = b;
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int k = 1; k < G; ++k) { a += sh[k * L + l]; b += sh[256 + k * L + l]; }
            }
            __syncthreads();                                 // the next round writes the sums again
        }
        if (e != 0.f) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { a[j] += e * bf2f(x[j]); b[j] += e * bf2f(x[4 + j]); }
        }
        bf16x8 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] = f2bf(a[j]); o[4 + j] = f2bf(b[j]); }
        if (ok) *reinterpret_cast<bf16x8*>(dh + (size_t)r * lddh + c * 8) = o;
    }
}

// dw (+)= scale (hi + lo)^T h for R <= 64 rows: hi, lo [R][ldp] bf16, the two parts of P.  A workgroup makes 64 entries x 256
// features: P's parts and h come into LDS whole (LDS-DMA; rows past R read as zeros), a wave takes 16 entries, and an MFMA's 64
// rows are all there is to contract: writing dw bounds it (32128 x 768: 49 MB, 9 us), but P's parts and h have to arrive whole first
// and it takes 17.4 us.  The MFMA's sixteen columns are taken as four
// fours, eight apart, so that two products leave a lane eight consecutive features of one entry: 16-byte stores.
constexpr int FEW = 64, FEW_P = 8192, FEW_H = 32768;
template <bool F32>
__global__ void __launch_bounds__(256) ce_dw_few_kernel(const bf16* __restrict__ hi, const bf16* __restrict__ lo, int ldp, const bf16* __restrict__ h, int ldh,
                                                        void* __restrict__ dw, int lddw, int R, int n, int d, float scale) {
    __shared__ __attribute__((aligned(16))) char smem[2 * FEW_P + FEW_H];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int v0 = blockIdx.x * 64, d0 = blockIdx.y * 256;
    const int cols = min(256, d - d0);                           // a multiple of 64
    const auto rh = __builtin_amdgcn_make_buffer_rsrc((void*)(hi + v0), 0, (uint32_t)(((size_t)(R - 1) * ldp + 64) * 2), 0x00020000);
    const auto rl = __builtin_amdgcn_make_buffer_rsrc((void*)(lo + v0), 0, (uint32_t)(((size_t)(R - 1) * ldp + 64) * 2), 0x00020000);
    const auto rx = __builtin_amdgcn_make_buffer_rsrc((void*)(h + d0), 0, (uint32_t)(((size_t)(R - 1) * ldh + cols) * 2), 0x00020000);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t off = stage_offset<true, 64>((i * 4 + w) * 64 + lane, ldp);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rh, LDS_PTR(smem + (i * 4 + w) * 1024), 16, off, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rl, LDS_PTR(smem + FEW_P + (i * 4 + w) * 1024), 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)                                  // (columns past d: a neighbour's values, not stored)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, LDS_PTR(smem + 2 * FEW_P + (i * 4 + w) * 1024), 16, stage_offset<true, 256>((i * 4 + w) * 64 + lane, ldh), 0, 0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    bf16x8 a[2][2];                                              // [part][32 rows]
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        a[0][kk] = read_frag<true, 64>(smem, w * 16, kk, lane);
        a[1][kk] = read_frag<true, 64>(smem + FEW_P, w * 16, kk, lane);
    }
    const int g = lane >> 4, i16 = lane & 15, q = i16 >> 2, piece = i16 & 3;
    const int hk = q | ((g & 1) << 2);
    const int v = v0 + w * 16 + i16;
    for (int nb = 0; nb < cols / 32; ++nb) {
        f32x4 acc[2] = {};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                // fragment of features nb * 32 + 8 piece + 4 b ..: rows kk * 32 + 8 g ..+7 (image of gemm_tiles.h, 256 columns)
                const char* at = smem + 2 * FEW_P + (kk * 32 + 8 * g + q) * 512 + (((nb * 2 + (piece >> 1)) ^ hk) << 5) + ((piece & 1) * 8 + b * 4) * 2;
                const bf16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)at);
                const bf16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(at + 4 * 512));
                const bf16x8 x = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
                acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, a[1][kk], acc[b], 0, 0, 0);
                acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, a[0][kk], acc[b], 0, 0, 0);
            }
        if (v >= n) continue;
        const int c = d0 + nb * 32 + g * 8;
        if (F32) {
            float* out = (float*)dw + (size_t)v * lddw + c;
#pragma unroll
            for (int b = 0; b < 2; ++b) *reinterpret_cast<f32x4*>(out + 4 * b) += acc[b] * scale;
        } else {
            const bf16x4 o0 = __builtin_convertvector(acc[0] * scale, bf16x4), o1 = __builtin_convertvector(acc[1] * scale, bf16x4);
            __builtin_nontemporal_store(__builtin_shufflevector(o0, o1, 0, 1, 2, 3, 4, 5, 6, 7), reinterpret_cast<bf16x8*>((bf16*)dw + (size_t)v * lddw + c));
        }
    }
}

int blocks_for(long long items) {
    const long long g = (items + 255) / 256;
    return (int)(g < 1 ? 1 : g > 16384 ? 16384 : g);
}

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

// Microseconds of a product of M x N in tiles of edge `tile`, `steps` K steps of 64 cut into `slices`, as fitted to 650 launches
// of gemm.hip's kernels at 40 sizes (off by 4 to 10 % in the mean): a launch, and for every round of the chip's compute units
// the K steps and what a tile costs beside them.  Kernels as launch_cfg chooses them: rings for one and two 128x128 tiles and
// up to three 64x64 tiles a compute unit, several workgroups with one buffer beyond.  (A plan asks it
// some hundred times: 2 us, 9 for several pieces.)
long long tiles_of(int tile, int M, int N) { return (long long)((M + tile - 1) / tile) * ((N + tile - 1) / tile); }
double product_us(int tile, long long items, int slices, int steps, int cus) {
    const double rounds = (double)((items + cus - 1) / cus), load = (double)items / cus, per = (double)((steps + slices - 1) / slices);
    const bool ring = per >= 3.;
    if (tile == 256) return 2.3 + rounds * (per * (1.35 + 0.3 * (load < 1. ? load : 1.)) + 5.7);
    if (tile == 128) {
        if (ring && items <= cus) return 5.5 + per * (0.55 + 0.14 * load);
        if (ring && items <= 2 * cus) return 5.0 + per * (0.51 + 0.245 * load);
        return 4.4 + rounds * (per * 0.65 + 2.3);
    }
    if (ring && items <= 3 * cus) return 5.0 + per * (items <= cus ? 0.33 : items <= 2 * cus ? 0.375 : 0.57);
    return 5.0 + (load < 1. ? 1. : load) * (per * 0.2 + 0.4);
}
double tile_us(int tile, int M, int N, int steps, int cus) { return product_us(tile, tiles_of(tile, M, N), 1, steps, cus); }
int best_tile(int M, int N, int steps, int cus) {
    double best = 1e30;
    int tile = 64;
    for (int t = 256; t >= 64; t /= 2) {
        if (t == 256 && (M < 256 || N < 256)) continue;
        const double us = tile_us(t, M, N, steps, cus);
        if (us < best) { best = us; tile = t; }
    }
    return tile;
}

// what a product in two launches takes beside them (32128 x 768 from 300 rows: by the launches alone 26 us against 30 for one,
// measured 32 against 28)
constexpr double TWO_LAUNCHES = 6.;
// of M x N 256x256 tiles, the rows that fill whole rounds of the compute units
int whole_rounds(int M, int N, int cus) {
    const int wide = (N + 255) / 256, a_round = cus / wide;
    return a_round ? M / 256 / a_round * a_round * 256 : 0;
}

// Tile and slices of dh's product over a piece: more slices give it more workgroups and its second kernel more slabs to add
// (written and read at about 7 TB/s).  Of 13 sizes measured with 6 to 18 plans each the best is chosen at 10, one 2 to 10 %
// behind at three.  1088 x 768 from 32128: 9 slices of 128x128 tiles 67 us, 17 of 256x256 68, 14 of 128x128 (three
// workgroups a compute unit) 99; 512 x 768 from 8704: 5 of 64x64 19, 8 of 128x128 22, 32 of 256x256 30.
double dh_us(int R, int d, int steps, int* tile, int* slices, int cus) {
    double best = 1e30;
    for (int t = 256; t >= 64; t /= 2) {
        if (t == 256 && (R < 256 || d < 256)) continue;
        const long long tiles = tiles_of(t, R, d);
        for (int s = 1; s <= 64 && s * 3 <= steps + 2; ++s) {
            const double us = product_us(t, tiles * s, s, steps, cus) + (double)s * R * d * 8. / 7e6;
            if (us < best) { best = us; *slices = s; *tile = t; }
            if (tiles * s > 4ll * cus) break;
        }
    }
    return best;
}

// Pieces of the vocabulary: P takes at most 256 MiB (256 columns at least), a piece of the weights 2 GiB (the products address
// a transposed operand with 32-bit byte offsets).  Where it takes several, sixteen widths between half and all of that are
// compared by their estimated times; a narrower one has to gain 3 % (8192 rows x 32128 x 768: 64 tiles 1234 us, 42 tiles, on a
// par by the estimate, 1270).
double dw_us(int n, int d, int steps, int cus, int* rows);
struct CePlan { int piece, ldp, slabs, dh_tile; };
CePlan ce_plan(int R, int V, int d) {
    const int cus = paced_cu_count();
    CePlan pl;
    long long fit = (256ll << 20) / 2 / (R > 0 ? R : 1) / 256;       // in tiles of 256 columns
    const long long reach = (1ll << 30) / d / 256;
    if (fit > reach) fit = reach;
    if (fit < 1) fit = 1;
    long long piece = fit * 256;
    if (piece >= V) piece = V;
    else {
        double best = 1e30;
        const long long down = fit / 32 > 0 ? fit / 32 : 1;
        for (long long c = fit; c >= 1 && c * 2 >= fit && c > fit - 16 * down; c -= down) {
            double us = 0.;
            const int full = (int)(V / (c * 256)), rest = (int)(V - full * c * 256), k = (R + 63) / 64;
            for (int part = 0; part < 2; ++part) {
                const int n = part ? rest : (int)c * 256;
                if (n == 0 || (!part && !full)) continue;
                int tile = 64, slices = 1, rows;
                us += (part ? 1 : full) * (tile_us(best_tile(R, n, d / 64, cus), R, n, d / 64, cus) + dh_us(R, d, (n + 63) / 64, &tile, &slices, cus) +
                                           dw_us(n, d, k, cus, &rows));
            }
            if (us < best * 0.97) { best = us; piece = c * 256; }
        }
    }
    pl.piece = (int)piece;
    pl.ldp = (int)((piece + 63) / 64 * 64);
    const int steps = (pl.piece + 63) / 64;
    pl.slabs = 1;
    pl.dh_tile = 64;
    dh_us(R, d, steps, &pl.dh_tile, &pl.slabs, cus);
    const int per = (steps + pl.slabs - 1) / pl.slabs;
    pl.slabs = (steps + per - 1) / per;
    return pl;
}

GemmParams product(const void* A, int lda, const void* B, int ldb, void* C, int ldc, int M, int N, int K, float alpha) {
    GemmParams p = {};
    p.A = (const bf16*)A; p.B = (const bf16*)B; p.C = C;
    p.M = M; p.N = N; p.K = K; p.lda = lda; p.ldb = ldb; p.ldc = ldc;
    p.k_per_split = K; p.batch = 1; p.alpha = alpha; p.mask_scale = 1.f; p.drop = make_drop(0.f, 0);
    return p;
}

// Tile of the logits' product where it goes out as one launch.  Up to 64 rows 64x64 tiles read the weights fastest (16 rows: 16.6 us
// against 18.4 with 128x128).  forced (0: none) is paced_gemm_set_tile's, read once by a call: its workspace's layout hangs on it.
int ce_tile(int R, int N, int steps, int cus, int forced) { return forced ? forced : R <= FEW ? 64 : best_tile(R, N, steps, cus); }

// rows or columns of the logits, and rows of dw, in the first of two launches of this thread's most recent products (0: one launch)
struct Split { int rows, cols, dw_rows; };
thread_local Split t_split = {0, 0, 0};

// One product of the logits (EPI_CE_STATS or EPI_CE_GRAD): in one launch, or in two, 256x256 tiles and what they leave over in
// 128x128 tiles, where that saves a round: the rows that fill tiles and the rest (1088 rows x 32128 entries: 3 rounds for 4.25
// tiles of rows, 2 for 4), or the columns that fill whole rounds and the rest (1000 x 50001: 3.06 rounds).  Both launches leave
// statistics of 64 columns.
int ce_logits(GemmParams p, int epilogue, int forced, hipStream_t s) {
    const int steps = (p.K + 63) / 64, R = p.M, full = R / 256 * 256, cus = paced_cu_count();
    p.tile = ce_tile(R, p.N, steps, cus, forced);
    GemmParams rest = p;
    double best = tile_us(p.tile, R, p.N, steps, cus);
    int rows = 0, cols = 0;                                      // of the first launch (0: one launch)
    if (full > 0 && p.N >= 256 && !forced) {                     // (64x64 tiles leave another width of statistics)
        if (full < R) {
            const double us = tile_us(256, full, p.N, steps, cus) + tile_us(128, R - full, p.N, steps, cus) + TWO_LAUNCHES;
            if (us < best) { best = us; rows = full; }
        }
        const int limit = p.grid_limit >= 0 ? p.grid_limit : paced_gemm_default_grid_limit();
        const int fill = whole_rounds(p.N, R, limit > 0 && limit < cus ? limit : cus);
        if (fill > 0 && fill < p.N && tile_us(256, R, fill, steps, cus) + tile_us(128, R, p.N - fill, steps, cus) + TWO_LAUNCHES < best) { rows = 0; cols = fill; }
    }
    t_split.rows = rows;
    t_split.cols = cols;
    if (!rows && !cols) return paced_gemm_launch(p, false, false, epilogue, 1, s);
    p.tile = 256;
    rest.tile = 128;
    if (rows) {
        p.M = rows;
        rest.M -= rows;
        rest.A += (size_t)rows * p.lda;
        rest.ce_labels += rows;
        if (epilogue == EPI_CE_STATS) { rest.ce_part += rows; rest.ce_target += rows; }
        else { rest.ce_lse += rows; rest.ce_g += rows; rest.ce_err += rows; if (p.ce_loss) rest.ce_loss += rows; rest.C = (bf16*)rest.C + (size_t)rows * p.ldc; }
    } else {
        p.N = cols;
        rest.N -= cols;
        rest.B += (size_t)cols * p.ldb;
        rest.ce_first += cols;
        if (epilogue == EPI_CE_STATS) rest.ce_part += (size_t)(cols / 64) * p.ce_rows;
        else rest.C = (bf16*)rest.C + cols;
    }
    const int rc = paced_gemm_launch(p, false, false, epilogue, 1, s);
    return rc != PACED_OK ? rc : paced_gemm_launch(rest, false, false, epilogue, 1, s);
}

// dw's product over a piece, rows of P^T split like the logits' columns (32128 x 768: 378 tiles of 256 in two rounds, or 255 in
// one and the rest in 128x128 tiles: from 4096 rows 424 us with the logits again, then 405; from 1088 both 133).
double dw_us(int n, int d, int steps, int cus, int* rows) {
    const double one = tile_us(best_tile(n, d, steps, cus), n, d, steps, cus);
    *rows = 0;
    const int fill = d >= 256 ? whole_rounds(n, d, cus) : 0;
    if (fill == 0 || fill >= n) return one;
    const double two = tile_us(256, fill, d, steps, cus) + tile_us(best_tile(n - fill, d, steps, cus), n - fill, d, steps, cus) + TWO_LAUNCHES;
    if (two >= one) return one;
    *rows = fill;
    return two;
}
int ce_dw(GemmParams p, int epilogue, size_t element, int forced, hipStream_t s) {
    const int steps = (p.K + 63) / 64, cus = paced_cu_count();
    int rows = 0;
    if (!forced) dw_us(p.M, p.N, steps, cus, &rows);
    t_split.dw_rows = rows;
    if (rows) {
        GemmParams first = p;
        first.M = rows;
        first.tile = 256;
        const int rc = paced_gemm_launch(first, true, true, epilogue, 1, s);
        if (rc != PACED_OK) return rc;
        p.M -= rows;
        p.A += rows;
        p.C = (char*)p.C + (size_t)rows * p.ldc * element;
    }
    p.tile = forced ? forced : best_tile(p.M, p.N, steps, cus);
    return paced_gemm_launch(p, true, true, epilogue, 1, s);
}

int ce_check(const char* who, const void* h, int ldh, const void* w, int ldw, const long long* labels, int R, int V, int d) {
    PACED_CHECK_ARG(R >= 0 && V > 0 && d > 0 && d % 64 == 0, "%s: need R >= 0, V > 0 and d a multiple of 64 (R=%d V=%d d=%d)", who, R, V, d);
    if (R == 0) return PACED_OK;
    PACED_CHECK_ARG(h && w && labels, "%s: null operand", who);
    PACED_CHECK_ARG(ldh >= d && ldw >= d && ldh % 8 == 0 && ldw % 8 == 0 && (((uintptr_t)h | (uintptr_t)w) & 15) == 0,
                    "%s: h and w need 16-byte aligned rows, strides of at least d and multiples of 8 (ldh=%d ldw=%d)", who, ldh, ldw);
    PACED_CHECK_ARG(ldh <= 1 << 22 && ldw <= 1 << 22, "%s: a tile of 256 rows must span less than 4 GiB: row strides up to 2^22 (ldh=%d ldw=%d)", who, ldh, ldw);
    return PACED_OK;
}

}  // namespace

extern "C" int paced_linear_ce_last_split(int* rows, int* cols, int* dw_rows) {
    PACED_CHECK_ARG(rows && cols && dw_rows, "paced_linear_ce_last_split: null operand");
    *rows = t_split.rows;
    *cols = t_split.cols;
    *dw_rows = t_split.dw_rows;
    return PACED_OK;
}

namespace {
size_t stats_bytes(int R, int V, int width) { return round256((size_t)((V + width - 1) / width) * R * 8); }
}  // namespace

// (any d, any forced tile)
extern "C" size_t paced_linear_ce_fwd_workspace_bytes(int R, int V) {
    if (R <= 0 || V <= 0) return 0;
    return stats_bytes(R, V, 32) + round256((size_t)R * 4);
}

// statistics of 32 columns come from 64x64 tiles alone, which only small products take
namespace {
size_t fwd_workspace(int R, int V, int d, int forced) {
    return stats_bytes(R, V, ce_tile(R, V, (d + 63) / 64, paced_cu_count(), forced) == 64 ? 32 : 64) + round256((size_t)R * 4);
}
}  // namespace
extern "C" size_t paced_linear_ce_fwd_workspace_bytes_for(int R, int V, int d) {
    return R <= 0 || V <= 0 || d <= 0 ? 0 : fwd_workspace(R, V, d, paced_gemm_forced_tile());
}

extern "C" int paced_linear_ce_fwd_ex(const void* h, int ldh, const void* w, int ldw, const long long* labels, float* loss, float* lse,
                                      int R, int V, int d, long long ignore_index, float scale, int grid_limit, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    const int rc = ce_check("paced_linear_ce_fwd", h, ldh, w, ldw, labels, R, V, d);
    if (rc != PACED_OK || R == 0) return rc;
    PACED_CHECK_ARG(loss, "paced_linear_ce_fwd: null operand");
    const int forced = paced_gemm_forced_tile();
    const size_t need = fwd_workspace(R, V, d, forced);
    PACED_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                    "paced_linear_ce_fwd: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need, workspace_bytes);
    GemmParams p = product(h, ldh, w, ldw, nullptr, 0, R, V, d, scale);
    p.ce_part = (f32x2*)workspace;
    p.ce_target = (float*)((char*)workspace + (need - round256((size_t)R * 4)));
    p.ce_labels = labels; p.ce_ignore = ignore_index; p.ce_vocab = V;
    p.ce_rows = R;
    p.grid_limit = grid_limit;
    const int rg = ce_logits(p, EPI_CE_STATS, forced, (hipStream_t)stream);
    if (rg != PACED_OK) return rg;
    const int width = paced_gemm_stat_width();
    const int groups = (V + width - 1) / width;
    if (R >= 2 * paced_cu_count())
        hipLaunchKernelGGL(ce_join_kernel<8>, dim3((R + 7) / 8), dim3(256), 0, (hipStream_t)stream, p.ce_part, groups, p.ce_target, labels, ignore_index, V, loss, lse, R);
    else
        hipLaunchKernelGGL(ce_join_kernel<1>, dim3(R), dim3(256), 0, (hipStream_t)stream, p.ce_part, groups, p.ce_target, labels, ignore_index, V, loss, lse, R);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}

extern "C" int paced_linear_ce_fwd(const void* h, int ldh, const void* w, int ldw, const long long* labels, float* loss, float* lse,
                                   int R, int V, int d, long long ignore_index, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    return paced_linear_ce_fwd_ex(h, ldh, w, ldw, labels, loss, lse, R, V, d, ignore_index, scale, -1, workspace, workspace_bytes, stream);
}

namespace {
size_t ce_workspace(const CePlan& pl, int R, int d) {
    return (R <= FEW ? 2 : 1) * round256((size_t)R * pl.ldp * 2) + round256((size_t)R * 4) + (size_t)pl.slabs * R * d * 4;
}
}  // namespace

extern "C" size_t paced_linear_ce_bwd_workspace_bytes(int R, int V, int d) {
    return R <= 0 || V <= 0 || d <= 0 ? 0 : ce_workspace(ce_plan(R, V, d), R, d);
}

extern "C" int paced_linear_ce_bwd_ex(const void* h, int ldh, const void* w, int ldw, const long long* labels, const float* loss, const float* lse,
                                      const float* gloss, void* dh, int lddh, void* dw, int lddw, int dw_f32, int R, int V, int d,
                                      long long ignore_index, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = ce_check("paced_linear_ce_bwd", h, ldh, w, ldw, labels, R, V, d);
    if (rc != PACED_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    PACED_CHECK_ARG(!dw || (lddw >= d && lddw % 8 == 0 && ((uintptr_t)dw & 15) == 0), "paced_linear_ce_bwd: dw needs 16-byte aligned rows, a stride of at least d and a multiple of 8 (lddw=%d)", lddw);
    if (R == 0) {                                     // no row: dw's sum is empty
        if (!dw || dw_f32) return PACED_OK;
        hipLaunchKernelGGL(ce_dh_kernel<1>, dim3(blocks_for((long long)V * (d >> 3))), dim3(256), 0, s, nullptr, 0, 0LL, (bf16*)dw, lddw, V, d,
                           nullptr, 0LL, 0, nullptr, nullptr, 0, 0.f);
        PACED_CHECK_LAUNCH();
        return PACED_OK;
    }
    PACED_CHECK_ARG(lse && gloss, "paced_linear_ce_bwd: null operand");
    PACED_CHECK_ARG(!dh || (lddh >= d && lddh % 8 == 0 && ((uintptr_t)dh & 15) == 0), "paced_linear_ce_bwd: dh needs 16-byte aligned rows, a stride of at least d and a multiple of 8 (lddh=%d)", lddh);
    CePlan pl = ce_plan(R, V, d);
    const size_t need = ce_workspace(pl, R, d);
    PACED_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                    "paced_linear_ce_bwd: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need, workspace_bytes);
    // a transposed operand is addressed with 32-bit byte offsets from its first row
    PACED_CHECK_ARG((unsigned long long)R * (ldh > pl.ldp ? ldh : pl.ldp) < (1ull << 31), "paced_linear_ce_bwd: %d rows of h with a stride of %d span 4 GiB or more; pass fewer at a time", R, ldh);
    // (of w only a piece: one whose rows lie so far apart that the plan's piece is out of reach goes by in narrower ones, which
    // need no more of the workspace: 256 rows at the largest stride)
    const int reach = (int)(((1u << 31) - 1) / (unsigned)ldw / 256 * 256);
    if (pl.piece > reach) {
        pl.piece = reach;
        pl.ldp = reach;
        const int steps = reach / 64, per = (steps + pl.slabs - 1) / pl.slabs;
        pl.slabs = (steps + per - 1) / per;                       // (the first piece writes every slab)
    }
    bf16* P = (bf16*)workspace;
    const size_t part = round256((size_t)R * pl.ldp * 2);
    t_split = Split{0, 0, 0};
    const int forced = paced_gemm_forced_tile();                  // (the low part is written by the 64x64 tiles' epilogue)
    bf16* low = dw && R <= FEW && (forced == 0 || forced == 64) ? (bf16*)((char*)workspace + part) : nullptr;
    float* err = (float*)((char*)workspace + (R <= FEW ? 2 : 1) * part);
    float* slabs = (float*)((char*)err + round256((size_t)R * 4));
    for (int v0 = 0; v0 < V; v0 += pl.piece) {
        const int n = V - v0 < pl.piece ? V - v0 : pl.piece;
        const bf16* wp = (const bf16*)w + (size_t)v0 * ldw;
        GemmParams p = product(h, ldh, wp, ldw, P, pl.ldp, R, n, d, scale);
        p.ce_labels = labels; p.ce_lse = lse; p.ce_g = gloss; p.ce_loss = loss;
        p.ce_ignore = ignore_index; p.ce_vocab = V; p.ce_first = v0;
        p.ce_err = err; p.ce_lo = low;
        int r = ce_logits(p, EPI_CE_GRAD, forced, s);
        if (r != PACED_OK) return r;
        if (dh) {
            p = product(P, pl.ldp, wp, ldw, slabs, d, R, d, n, scale);
            p.strideC = (long long)R * d;
            p.accumulate = v0 > 0;
            p.tile = forced ? forced : pl.dh_tile;
            if ((r = paced_gemm_launch(p, false, true, EPI_SLAB_F32, pl.slabs, s)) != PACED_OK) return r;
        }
        if (dw && low) {
            const dim3 grid((n + 63) / 64, (d + 255) / 256);
            if (dw_f32) hipLaunchKernelGGL(ce_dw_few_kernel<true>, grid, dim3(256), 0, s, P, low, pl.ldp, (const bf16*)h, ldh, (void*)((float*)dw + (size_t)v0 * lddw), lddw, R, n, d, scale);
            else hipLaunchKernelGGL(ce_dw_few_kernel<false>, grid, dim3(256), 0, s, P, low, pl.ldp, (const bf16*)h, ldh, (void*)((bf16*)dw + (size_t)v0 * lddw), lddw, R, n, d, scale);
            PACED_CHECK_LAUNCH();
        } else if (dw) {
            p = product(P, pl.ldp, h, ldh, dw_f32 ? (void*)((float*)dw + (size_t)v0 * lddw) : (void*)((bf16*)dw + (size_t)v0 * lddw), lddw, n, d, R, scale);
            p.accumulate = 1;
            if ((r = ce_dw(p, dw_f32 ? EPI_SLAB_F32 : EPI_BF16, dw_f32 ? 4 : 2, forced, s)) != PACED_OK) return r;
        }
    }
    if (dh) {
        const long long pieces = (long long)R * (d >> 3);
        if (pieces < 256LL * paced_cu_count())
            hipLaunchKernelGGL(ce_dh_kernel<8>, dim3(blocks_for(pieces * 8)), dim3(256), 0, s, slabs, pl.slabs, (long long)R * d, (bf16*)dh, lddh, R, d,
                               labels, ignore_index, V, err, (const bf16*)w, ldw, scale);
        else
            hipLaunchKernelGGL(ce_dh_kernel<1>, dim3(blocks_for(pieces)), dim3(256), 0, s, slabs, pl.slabs, (long long)R * d, (bf16*)dh, lddh, R, d,
                               labels, ignore_index, V, err, (const bf16*)w, ldw, scale);
        PACED_CHECK_LAUNCH();
    }
    return PACED_OK;
}

extern "C" int paced_linear_ce_bwd(const void* h, int ldh, const void* w, int ldw, const long long* labels, const float* lse, const float* gloss,
                                   void* dh, int lddh, void* dw, int lddw, int dw_f32, int R, int V, int d, long long ignore_index, float scale,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    return paced_linear_ce_bwd_ex(h, ldh, w, ldw, labels, nullptr, lse, gloss, dh, lddh, dw, lddw, dw_f32, R, V, d, ignore_index, scale,
                                  workspace, workspace_bytes, stream);
}
