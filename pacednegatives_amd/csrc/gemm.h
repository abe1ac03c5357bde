// Internal interface of the tiled bf16 MFMA contraction kernel (gemm.hip).
#pragma once
#include "common.h"

enum Epi : int {
    EPI_BF16 = 0,        // C = acc
    EPI_RES_DROP = 1,    // C = aux + dropout(acc)
    EPI_RELU_DROP = 2,   // C = dropout(relu(acc)); if aux: bit (m, n) of the byte matrix aux = (C > 0)
    EPI_MASK = 3,        // C = acc * (aux > 0 ? mask_scale : 0)
    EPI_F32 = 4,         // C(f32) = acc
    EPI_ATOMIC_F32 = 5,  // C(f32) += acc   (atomic, split-K allowed)
    EPI_MASK_BITS = 6,   // C = acc * (bit (m, n) of the byte matrix aux ? mask_scale : 0)
    EPI_COUNT,           // ---- epilogues below are internal to the pool scorer (mining.hip)
    EPI_TOPK_DENSE = 7,  // cand[n][m] = key(acc, row_base + m)
    EPI_TOPK_FILTER = 8, // if acc >= thr[n]: cand[n][cnt[n]++] = key(acc, row_base + m)
    // ---- internal to the linear-head cross entropy (linear_ce.hip); rows m are tokens, columns n vocabulary entries
    EPI_CE_STATS = 9,    // part[n / W * ce_rows + m] = (max, sum of 2^(z - max)) of z = acc * alpha * log2 e over W columns but the label's
                         // (W = paced_gemm_stat_width(), 32 or 64); target[m] = the label's acc * alpha
    EPI_CE_GRAD = 10,    // C(bf16) = g[m] 2^(z - lse[m] log2 e), the label's g[m] (exp(-loss[m]) - 1); columns N .. next multiple of 64 are zeros
    EPI_SLAB_F32 = 11    // C(f32) + split * strideC elements (+)= acc * alpha: one owner per element, no atomics
};

// Every field has a value from the start: a launch reads fields (tile, accumulate, ce_*) that most callers never set.
struct GemmParams {
    const bf16* A = nullptr;
    const bf16* B = nullptr;
    void* C = nullptr;
    const bf16* aux = nullptr;
    int M = 0, N = 0, K = 0;
    int lda = 0, ldb = 0, ldc = 0, ldaux = 0;
    int k_per_split = 0;   // multiple of BK
    // Head-major operands (> 0: elements between heads; the operand's leading dimension is then 64): the operand's feature
    // columns [64h, 64h + 64) are the contiguous [rows, 64] matrix at base + h * stride instead of a column block of rows of
    // ld elements.  A: features = K (not transposed) or M (transposed); B: transposed only, features = N; C: plain bf16
    // epilogue only, features = N.
    long long a_heads = 0, b_heads = 0, c_heads = 0;
    int batch = 1;         // independent problems of the same shape; operand b starts strideX * b elements after operand 0
    long long strideA = 0, strideB = 0, strideC = 0;
    float alpha = 1.f;     // scales acc before the epilogue
    float mask_scale = 1.f;
    DropCfg drop = {};
    int drop_narrow = 0;   // the output has at most 2^34 elements: dropout's quad numbers fit 32 bits
    // pool scorer only
    unsigned long long* tk_cand = nullptr;
    unsigned int* tk_cnt = nullptr;
    const float* tk_thr = nullptr;
    int tk_cap = 0;
    unsigned int tk_row_base = 0;
    // linear-head cross entropy only
    const long long* ce_labels = nullptr;   // [M]; a label counts when it is not ce_ignore and lies in [0, ce_vocab)
    const float* ce_lse = nullptr;          // [M]
    const float* ce_g = nullptr;            // [M]
    const float* ce_loss = nullptr;         // [M] (NULL: the label's entry is made from ce_lse)
    float* ce_err = nullptr;                // [M] EPI_CE_GRAD: what the label's entry lost in its rounding (rows with a label among the columns)
    bf16* ce_lo = nullptr;                  // EPI_CE_GRAD, small tiles: what every entry lost, in bf16, laid out as C (NULL: not wanted)
    f32x2* ce_part = nullptr;
    float* ce_target = nullptr;
    long long ce_ignore = 0;
    int ce_vocab = 0, ce_first = 0;         // vocabulary size, entry of column 0
    int ce_rows = 0;                        // rows of part (a launch may cover some of them)
    int accumulate = 0;                     // EPI_SLAB_F32: add to what is there
    int tile = 0;                           // tile edge the caller has chosen (0: the launch's own rule, or paced_gemm_set_tile's)
    int grid_limit = -1;                    // most workgroups of a phased launch (< 0: the call's or the process's own; 0: one to a compute unit)
};

// Order-preserving 64-bit key: larger key <=> (higher score, then lower pool row).
__host__ __device__ __forceinline__ unsigned long long topk_key(float score, unsigned int row) {
    score += 0.0f;                                   // -0 -> +0
    unsigned int u = __builtin_bit_cast(unsigned int, score);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (unsigned long long)(~row);
}
__host__ __device__ __forceinline__ float topk_key_score(unsigned long long key) {
    unsigned int u = (unsigned int)(key >> 32);
    u = (u & 0x80000000u) ? (u & 0x7fffffffu) : ~u;
    return __builtin_bit_cast(float, u);
}
__host__ __device__ __forceinline__ unsigned int topk_key_row(unsigned long long key) { return ~(unsigned int)key; }

// Launches the tiled kernel for (trans_a, trans_b, epilogue); arguments are already validated.
// tile edge that paced_gemm_set_tile has forced (0: none)
int paced_gemm_forced_tile();
// most workgroups of a phased launch where GemmParams names no limit (0: one to a compute unit)
int paced_gemm_default_grid_limit();
// columns per statistics group of the calling thread's most recent EPI_CE_STATS launch
int paced_gemm_stat_width();
int paced_gemm_launch(const GemmParams& p, bool trans_a, bool trans_b, int epilogue, int splits, hipStream_t stream);



// Pool scoring for at most 128 queries with the HBM-streaming kernel (EPI_TOPK_FILTER's contract: p.A pool rows [M, K],
// p.B queries [N, K], p.tk_*); PACED_ERR_ARG when the shape is outside what it covers (the caller then takes the tiled kernel).
int paced_pool_stream_launch(const GemmParams& p, hipStream_t stream);
