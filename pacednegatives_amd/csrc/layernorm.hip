// Layer norm, forward and backward, with an optional residual sum in front of it and the reduction of the weight's and the
// bias's gradient:
//   s = x (+ res, rounded to the tensors' type: it is what the backward pass reads)      xsum = s
//   mean = sum(s) / d     rstd = 1 / sqrt(sum((s - mean)^2) / d + eps)     y = (s - mean) rstd w + b
//   xh = (s - mean) rstd    g = dy w    dx = rstd (g - sum(g) / d - xh sum(g xh) / d) (+ dres)
//   dw += sum over rows of dy xh        db += sum over rows of dy
// Bound by memory: every stream is read or written once.  A TEAM of threads holds a whole row in registers, so the mean, the
// squares about it and the output take one read of the row; statistics and sums are 32-bit.  Column sums stay in registers
// over all rows that a team works on, are added over a workgroup's teams in LDS, and leave as one partial row per workgroup;
// a second kernel adds those in a fixed order (no atomics: equal inputs give equal bits).
// Measured, 139264 x 768 bf16 with the residual sum: forward 150 us for its four streams (5.7 TB/s; a copy of 256 MB reaches
// 5.4), backward 167 to 173 us for its four (5.0 to 5.1 TB/s), column sums 4.7 us.  139264 x 767 (fp32, no residual): 166 and
// 258 us against 147 and 226 for 768.  5001 x 1023 fp32: 11, 18 and 4.5 us.
#include "common.h"

namespace {

constexpr int LN_BLOCK = 256;
constexpr int LN_MAX_D = 8192;

// 16 bytes of a row in a register quad.  The vector types carry the element's alignment only: gfx950 loads and stores 16 bytes
// at any element address, so rows of odd width or stride take the same path (single elements instead: 23 us for the backward
// pass of 5001 x 1023 fp32).  down(n): element n becomes the first, zeros follow the last.  store_first(n): the first n alone.
template <class T> struct Piece;
template <> struct Piece<bf16> {
    static constexpr int V = 8;
    typedef u32x4 __attribute__((aligned(2))) At;
    u32x4 r;
    __device__ __forceinline__ float get(int j) const { return __uint_as_float((j & 1) ? (r[j >> 1] & 0xffff0000u) : (r[j >> 1] << 16)); }
    __device__ __forceinline__ void put(const float (&f)[8]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bf16x2 v = {f2bf(f[2 * j]), f2bf(f[2 * j + 1])};
            r[j] = __builtin_bit_cast(uint32_t, v);
        }
    }
    __device__ __forceinline__ void put_one(int j, bf16 x) {
        const uint32_t u = __builtin_bit_cast(unsigned short, x);
        r[j >> 1] = (j & 1) ? (r[j >> 1] & 0xffffu) | (u << 16) : (r[j >> 1] & 0xffff0000u) | u;
    }
    __device__ __forceinline__ bf16 one(int j) const { return __builtin_bit_cast(bf16, (unsigned short)(r[j >> 1] >> (16 * (j & 1)))); }
    __device__ __forceinline__ void down(int n) {
        if (n & 4) r = u32x4{r[2], r[3], 0u, 0u};
        if (n & 2) r = u32x4{r[1], r[2], r[3], 0u};
        if (n & 1) r = u32x4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
    }
    __device__ __forceinline__ void store_first(int n, bf16* at) const {
        typedef u32x2 __attribute__((aligned(2))) At4;
        typedef uint32_t __attribute__((aligned(2))) At2;
        u32x4 v = r;
        if (n & 4) { *reinterpret_cast<At4*>(at) = u32x2{v[0], v[1]}; v = u32x4{v[2], v[3], 0u, 0u}; at += 4; }
        if (n & 2) { *reinterpret_cast<At2*>(at) = v[0]; v[0] = v[1]; at += 2; }
        if (n & 1) *at = __builtin_bit_cast(bf16, (unsigned short)v[0]);
    }
};
template <> struct Piece<float> {
    static constexpr int V = 4;
    typedef f32x4 __attribute__((aligned(4))) At;
    f32x4 r;
    __device__ __forceinline__ float get(int j) const { return r[j]; }
    __device__ __forceinline__ void put(const float (&f)[4]) { r = f32x4{f[0], f[1], f[2], f[3]}; }
    __device__ __forceinline__ void put_one(int j, float x) { r[j] = x; }
    __device__ __forceinline__ float one(int j) const { return r[j]; }
    __device__ __forceinline__ void down(int n) {
        if (n & 2) r = f32x4{r[2], r[3], 0.f, 0.f};
        if (n & 1) r = f32x4{r[1], r[2], r[3], 0.f};
    }
    __device__ __forceinline__ void store_first(int n, float* at) const {
        typedef f32x2 __attribute__((aligned(4))) At2;
        f32x4 v = r;
        if (n & 2) { *reinterpret_cast<At2*>(at) = f32x2{v[0], v[1]}; v[0] = v[2]; at += 2; }
        if (n & 1) *at = v[0];
    }
};
// How a row ends.  FITS: with a whole piece.  LAPS: inside its last piece, which is loaded whole from d - V on and moved down by
// `settle` when all loads are on their way (single elements, each waited for: 139264 x 767 bf16 forward 144 us, backward 311).
// SHORT: the row is shorter than a piece; single elements.  Elements past the end are zeros.
enum End : int { FITS, LAPS, SHORT };
// STREAM: read once, past the caches
template <bool STREAM, End END, class T>
__device__ __forceinline__ void load_piece(Piece<T>& p, const T* row, int c, int d) {
    typedef typename Piece<T>::At At;
    p.r = decltype(p.r){};
    if (END == SHORT) {
#pragma unroll
        for (int j = 0; j < Piece<T>::V; ++j) if (c + j < d) p.put_one(j, row[c + j]);
    } else if (c < d) {
        const At* at = reinterpret_cast<const At*>(row + (END == LAPS ? min(c, d - Piece<T>::V) : c));
        p.r = STREAM ? __builtin_nontemporal_load(at) : *at;
    }
}
template <End END, class T>
__device__ __forceinline__ void settle(Piece<T>& p, int c, int d) {
    if (END == LAPS && c < d && c + Piece<T>::V > d) p.down(Piece<T>::V - d % Piece<T>::V);
}
template <End END, class T>
__device__ __forceinline__ void store_piece(const Piece<T>& p, T* row, int c, int d) {
    typedef typename Piece<T>::At At;
    if (END == SHORT) {
#pragma unroll
        for (int j = 0; j < Piece<T>::V; ++j) if (c + j < d) row[c + j] = p.one(j);
    } else if (END == FITS || c + Piece<T>::V <= d) {
        if (c < d) {
            // past the caches, but for bf16 rows at odd addresses, whose pieces share lines (139264 x 767: forward 108 us against
            // 114, backward 167 against 187; fp32 the other way, 168 against 166 and 270 against 266)
            if (END == LAPS && sizeof(T) == 2) *reinterpret_cast<At*>(row + c) = p.r;
            else __builtin_nontemporal_store(p.r, reinterpret_cast<At*>(row + c));
        }
    } else if (c < d) p.store_first(d % Piece<T>::V, row + c);
}

// sum over the TEAM threads of a row (16 or 64 lanes of a wave, or the whole workgroup through `sh`, two sets of four slots)
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* sh) {
#pragma unroll
    for (int o = (TEAM < 64 ? TEAM : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        v = sh[0] + sh[1] + sh[2] + sh[3];
    }
    return v;
}

template <class T> struct LnFwd {
    const T *x, *res, *w, *b;
    T *xsum, *y;
    float *mean, *rstd;
    int ldx, ldr, lds, ldy, M, d;
    float eps;
};

// (w and b are requested together with the row: behind the row's sums, from the caches, 1 x 768 took 5.2 us instead of 4.7,
// 4000 x 768 8.0 instead of 7.2, 139264 x 768 the same 148)
template <class T, int TEAM, int PER, End END>
__global__ void __launch_bounds__(LN_BLOCK) ln_fwd_kernel(LnFwd<T> a) {
    constexpr int V = Piece<T>::V, RPB = LN_BLOCK / TEAM;
    __shared__ float sh[4][4];
    const int l = threadIdx.x % TEAM, t = threadIdx.x / TEAM;
    const float inv_d = 1.f / (float)a.d;
    const int last = a.d % V;                               // elements of a last piece that the row ends inside
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.M; row0 += (long long)gridDim.x * RPB) {
        const bool ok = row0 + t < a.M;
        const size_t row = ok ? row0 + t : a.M - 1;         // a team past the end repeats the last row and stores nothing
        Piece<T> p[PER], q[PER], w[PER], b[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            load_piece<true, END>(p[i], a.x + row * a.ldx, c, a.d);
            if (a.res) load_piece<true, END>(q[i], a.res + row * a.ldr, c, a.d);
            load_piece<false, END>(w[i], a.w, c, a.d);
            load_piece<false, END>(b[i], a.b, c, a.d);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            settle<END>(p[i], c, a.d);
            settle<END>(w[i], c, a.d);
            settle<END>(b[i], c, a.d);
            if (a.res) {
                settle<END>(q[i], c, a.d);
                float f[V];
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = p[i].get(j) + q[i].get(j);
                p[i].put(f);
                if (END != LAPS && ok) store_piece<END>(p[i], a.xsum + row * a.lds, c, a.d);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum += p[i].get(j);
        }
        const float mean = team_sum<TEAM>(sum, sh[0]) * inv_d;
        if (END == LAPS && a.res && ok)                     // (xsum may be res: behind the sum, when pieces that lap have been read)
#pragma unroll
            for (int i = 0; i < PER; ++i) store_piece<END>(p[i], a.xsum + row * a.lds, (l + i * TEAM) * V, a.d);
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            if (END == FITS ? c < a.d : c + V <= a.d) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float f = p[i].get(j) - mean;
                    sq += f * f;
                }
            } else if (END != FITS && c < a.d) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float f = j < last ? p[i].get(j) - mean : 0.f;
                    sq += f * f;
                }
            }
        }
        const float rstd = 1.f / sqrtf(team_sum<TEAM>(sq, sh[1]) * inv_d + a.eps);
        if (l == 0 && ok) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            Piece<T> o;
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = (p[i].get(j) - mean) * rstd * w[i].get(j) + b[i].get(j);
            o.put(f);
            if (ok) store_piece<END>(o, a.y + row * a.ldy, c, a.d);
        }
        if (TEAM > 64) __syncthreads();                     // the next row's sums reuse `sh`
    }
}

template <class T> struct LnBwd {
    const T *dy, *x, *w, *dres;
    const float *mean, *rstd;
    T* dx;
    float* part;                    // [gridDim.x][2][d]: sums of dy xh, then of dy; NULL: no column sums
    float *dw, *db;
    int lddy, ldx, ldr, lddx, M, d;
};

// two waves per SIMD: a thread carries its pieces of three rows and two column sums in up to 256 registers (one wave and 512
// for fp32 rows of more than 4096)
template <class T, int TEAM, int PER, End END>
__global__ void __launch_bounds__(LN_BLOCK) __attribute__((amdgpu_waves_per_eu(PER < 8 ? 2 : 1)))
ln_bwd_kernel(LnBwd<T> a) {
    constexpr int V = Piece<T>::V, RPB = LN_BLOCK / TEAM;
    __shared__ float sh[4][4];
    extern __shared__ float cols[];                         // [4 waves][d]
    const int l = threadIdx.x % TEAM, t = threadIdx.x / TEAM;
    const float inv_d = 1.f / (float)a.d;
    float sw[PER][V], sb[PER][V];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) sw[i][j] = sb[i][j] = 0.f;
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < a.M; row0 += (long long)gridDim.x * RPB) {
        const bool ok = row0 + t < a.M;
        const size_t row = ok ? row0 + t : a.M - 1;
        Piece<T> p[PER], q[PER], r[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            load_piece<true, END>(p[i], a.dy + row * a.lddy, c, a.d);
            load_piece<true, END>(q[i], a.x + row * a.ldx, c, a.d);
            r[i].r = decltype(r[i].r){};
            if (a.dres) load_piece<true, END>(r[i], a.dres + row * a.ldr, c, a.d);
        }
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sg = 0.f, sgx = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            if (c < a.d) {                                  // (past the end of a row dy and w are zeros)
                Piece<T> w;
                load_piece<false, END>(w, a.w, c, a.d);
                settle<END>(p[i], c, a.d);
                settle<END>(q[i], c, a.d);
                settle<END>(w, c, a.d);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float dy = p[i].get(j), xh = (q[i].get(j) - mean) * rstd, g = dy * w.get(j);
                    sg += g;
                    sgx += g * xh;
                    if (ok) { sw[i][j] += dy * xh; sb[i][j] += dy; }
                }
            }
        }
        sg = team_sum<TEAM>(sg, sh[0]) * inv_d;
        sgx = team_sum<TEAM>(sgx, sh[1]) * inv_d;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = (l + i * TEAM) * V;
            Piece<T> w, o;
            load_piece<false, END>(w, a.w, c, a.d);
            settle<END>(r[i], c, a.d);
            settle<END>(w, c, a.d);
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (q[i].get(j) - mean) * rstd;
                f[j] = rstd * (p[i].get(j) * w.get(j) - sg - xh * sgx) + r[i].get(j);
            }
            o.put(f);
            if (ok) store_piece<END>(o, a.dx + row * a.lddx, c, a.d);
        }
        if (TEAM > 64) __syncthreads();
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * 2 * a.d;
    if (TEAM >= LN_BLOCK) {                                 // one team: its registers are the workgroup's sums
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = (l + i * TEAM) * V + j;
                if (c < a.d) { out[c] = sw[i][j]; out[a.d + c] = sb[i][j]; }
            }
        return;
    }
    // teams of one wave first (lanes that hold the same columns), then the four waves through LDS, in a fixed order; the two
    // sums one after the other in the same LDS
    const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float u = k ? sb[i][j] : sw[i][j];
#pragma unroll
                for (int o = TEAM; o < 64; o <<= 1) u += __shfl_xor(u, o, 64);
                const int c = (l + i * TEAM) * V + j;
                if (lane < TEAM && c < a.d) cols[wv * a.d + c] = u;
            }
        __syncthreads();
        for (int c = threadIdx.x; c < a.d; c += LN_BLOCK)
            out[k * a.d + c] = (cols[c] + cols[a.d + c]) + (cols[2 * a.d + c] + cols[3 * a.d + c]);
        __syncthreads();
    }
}

// dw[c] += sum over g of part[g][0][c], db[c] += ... [1][c]: 32 columns of a workgroup, 32 threads over the partial rows of each
// (8 threads and one load at a time measured 20 us on 512 rows of 1536 columns)
constexpr int COLS_LANES = 32;
__global__ void __launch_bounds__(32 * COLS_LANES) ln_cols_kernel(const float* __restrict__ part, int G, int d, float* dw, float* db) {
    __shared__ float sh[COLS_LANES][33];
    const int l = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + l;
    float s = 0.f;
    if (c < 2 * d) {
        int g = k;
        for (; g + 3 * COLS_LANES < G; g += 4 * COLS_LANES) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = part[(size_t)(g + i * COLS_LANES) * 2 * d + c];
#pragma unroll
            for (int i = 0; i < 4; ++i) s += v[i];
        }
        for (; g < G; g += COLS_LANES) s += part[(size_t)g * 2 * d + c];
    }
    sh[k][l] = s;
    __syncthreads();
    // column l's lanes now side by side: lane k of the wave half adds slot k, five levels
    float t = sh[l][k];                              // transposed: this thread's column is k, its slot l
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    const int cc = blockIdx.x * 32 + k;
    if (l == 0 && cc < 2 * d) {
        if (cc < d) { if (dw) dw[cc] += t; }
        else if (db) db[cc - d] += t;
    }
}

constexpr int LN_BWD_PER_CU = 4;           // most workgroups of the backward kernel for a compute unit (the workspace's rows)

template <class T, int TEAM, int PER, End END>
int ln_go(const LnFwd<T>& a, hipStream_t s) {
    const long long blocks = ((long long)a.M + LN_BLOCK / TEAM - 1) / (LN_BLOCK / TEAM);
    const int grid = (int)(blocks < 8192 ? blocks : 8192);
    hipLaunchKernelGGL((ln_fwd_kernel<T, TEAM, PER, END>), dim3(grid), dim3(LN_BLOCK), 0, s, a);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}
template <class T, int TEAM, int PER, End END>
int ln_go(const LnBwd<T>& a, hipStream_t s) {
    // resident workgroups: up to 16 elements a thread need at most 128 registers, four to a compute unit; more need up to 256
    const int most = (PER * Piece<T>::V <= 16 ? LN_BWD_PER_CU : 2) * paced_cu_count();
    const long long rounds_of = ((long long)a.M + LN_BLOCK / TEAM - 1) / (LN_BLOCK / TEAM), rounds = (rounds_of + most - 1) / most;
    const int grid = (int)((rounds_of + rounds - 1) / rounds);          // every workgroup the same number of row groups
    const int smem = TEAM < LN_BLOCK && a.part ? 4 * a.d * 4 : 0;              // 32 KiB at most: these teams take d <= 2048
    hipLaunchKernelGGL((ln_bwd_kernel<T, TEAM, PER, END>), dim3(grid), dim3(LN_BLOCK), smem, s, a);
    PACED_CHECK_LAUNCH();
    if (!a.part) return PACED_OK;
    hipLaunchKernelGGL(ln_cols_kernel, dim3((2 * a.d + 31) / 32), dim3(32 * COLS_LANES), 0, s, a.part, grid, a.d, a.dw, a.db);
    PACED_CHECK_LAUNCH();
    return PACED_OK;
}

// the narrowest team whose registers hold a row of d elements
template <class T, End END, class Args>
int ln_team(const Args& a, hipStream_t s) {
    const int n = (a.d + Piece<T>::V - 1) / Piece<T>::V;     // pieces of a row
    if (n <= 16) return ln_go<T, 16, 1, END>(a, s);
    if constexpr (END != SHORT) {
        if (n <= 32) return ln_go<T, 16, 2, END>(a, s);
        if (n <= 64) return ln_go<T, 16, 4, END>(a, s);
        if (n <= 96) return ln_go<T, 16, 6, END>(a, s);
        if (n <= 128) return ln_go<T, 64, 2, END>(a, s);
        if (n <= 256) return ln_go<T, 64, 4, END>(a, s);
        if (n <= 512) return ln_go<T, 256, 2, END>(a, s);
        if (n <= 1024) return ln_go<T, 256, 4, END>(a, s);
        if constexpr (Piece<T>::V * 1024 < LN_MAX_D) return ln_go<T, 256, 8, END>(a, s);
    }
    return PACED_ERR_ARG;                                    // (d <= LN_MAX_D was checked)
}
template <class T, class Args>
int ln_launch(const Args& a, hipStream_t s) {
    static_assert(1024 * Piece<bf16>::V >= LN_MAX_D && 2048 * Piece<float>::V >= LN_MAX_D, "the widest teams hold the widest row");
    return a.d < Piece<T>::V ? ln_team<T, SHORT>(a, s) : a.d % Piece<T>::V ? ln_team<T, LAPS>(a, s) : ln_team<T, FITS>(a, s);
}

template <class T>
int ln_fwd(const void* x, int ldx, const void* res, int ldr, void* xsum, int lds, const void* w, const void* b, void* y, int ldy,
           float* mean, float* rstd, int M, int d, float eps, hipStream_t s) {
    return ln_launch<T>(LnFwd<T>{(const T*)x, (const T*)res, (const T*)w, (const T*)b, (T*)xsum, (T*)y, mean, rstd, ldx, ldr, lds, ldy, M, d, eps}, s);
}
template <class T>
int ln_bwd(const void* dy, int lddy, const void* x, int ldx, const void* w, const float* mean, const float* rstd, const void* dres, int ldr,
           void* dx, int lddx, float* dw, float* db, float* part, int M, int d, hipStream_t s) {
    return ln_launch<T>(LnBwd<T>{(const T*)dy, (const T*)x, (const T*)w, (const T*)dres, mean, rstd, (T*)dx, part, dw, db, lddy, ldx, ldr, lddx, M, d}, s);
}

}  // namespace

extern "C" int paced_layernorm_max_width(void) { return LN_MAX_D; }

extern "C" int paced_layernorm_fwd(const void* x, int ldx, const void* res, int ldr, void* xsum, int lds, const void* w, const void* b,
                                   void* y, int ldy, float* mean, float* rstd, int M, int d, int f32, float eps, void* stream) {
    PACED_CHECK_ARG(M >= 0 && d > 0 && d <= LN_MAX_D, "paced_layernorm_fwd: need M >= 0 and d in [1, %d] (M=%d d=%d)", LN_MAX_D, M, d);
    if (M == 0) return PACED_OK;
    PACED_CHECK_ARG(x && w && b && y, "paced_layernorm_fwd: null operand");
    PACED_CHECK_ARG((res == nullptr) == (xsum == nullptr), "paced_layernorm_fwd: res and xsum go together");
    PACED_CHECK_ARG(ldx >= d && ldy >= d && (!res || (ldr >= d && lds >= d)), "paced_layernorm_fwd: row strides must be at least d");
    PACED_CHECK_ARG(eps >= 0.f, "paced_layernorm_fwd: eps must not be negative");
    return f32 ? ln_fwd<float>(x, ldx, res, ldr, xsum, lds, w, b, y, ldy, mean, rstd, M, d, eps, (hipStream_t)stream)
               : ln_fwd<bf16>(x, ldx, res, ldr, xsum, lds, w, b, y, ldy, mean, rstd, M, d, eps, (hipStream_t)stream);
}

extern "C" size_t paced_layernorm_workspace_bytes(int M, int d) {
    if (M <= 0 || d <= 0) return 0;
    const size_t most = (size_t)LN_BWD_PER_CU * paced_cu_count();
    return ((size_t)M < most ? (size_t)M : most) * 2 * (size_t)d * 4;
}

extern "C" int paced_layernorm_bwd(const void* dy, int lddy, const void* x, int ldx, const void* w, const float* mean, const float* rstd,
                                   const void* dres, int ldr, void* dx, int lddx, float* dw, float* db, int M, int d, int f32,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    PACED_CHECK_ARG(M >= 0 && d > 0 && d <= LN_MAX_D, "paced_layernorm_bwd: need M >= 0 and d in [1, %d] (M=%d d=%d)", LN_MAX_D, M, d);
    if (M == 0) return PACED_OK;
    PACED_CHECK_ARG(dy && x && w && mean && rstd && dx, "paced_layernorm_bwd: null operand");
    PACED_CHECK_ARG(lddy >= d && ldx >= d && lddx >= d && (!dres || ldr >= d), "paced_layernorm_bwd: row strides must be at least d");
    const bool sums = dw || db;
    const size_t need = sums ? paced_layernorm_workspace_bytes(M, d) : 0;
    PACED_CHECK_ARG(!sums || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0),
                    "paced_layernorm_bwd: the column sums need a workspace of %zu bytes, got %zu", need, workspace_bytes);
    float* part = sums ? (float*)workspace : nullptr;
    return f32 ? ln_bwd<float>(dy, lddy, x, ldx, w, mean, rstd, dres, ldr, dx, lddx, dw, db, part, M, d, (hipStream_t)stream)
               : ln_bwd<bf16>(dy, lddy, x, ldx, w, mean, rstd, dres, ldr, dx, lddx, dw, db, part, M, d, (hipStream_t)stream);
}
