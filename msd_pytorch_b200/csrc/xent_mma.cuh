// The tensor-core products of the linear layer with softmax cross entropy (xent.h): one
// persistent kernel template with three uses.
//
//   kLse    z tile = x W^T, epilogue: per token the maximum and sum of exp over the tile's labels
//   kGrad   the same product again, epilogue: G = exp(z - lse) - onehot, rounded to 16 bits, stored
//   kBack   dx = G W and dW = G^T x: two lists of tiles in one launch, longest first
//
// Operands are 16-bit: bfloat16 and float16 inputs as they are, float32 inputs as the sum of three
// bfloat16 pieces v = a + b + c of 8 bits each (round to nearest: |b| <= 2^-9 |v|, |c| <= 2^-18 |v|, and
// 2^-27 |v| is left).  A product is a a' + (a b' + b a') + (a c' + b b' + c a'): what is dropped is below
// 2^-25 of it, less than a float32 product's own rounding, and as the pieces have float32's range of exponents
// this holds whatever the other values of the tensor are.  (Two float16 pieces under one power of two
// per tensor need three products instead of six, but hold nothing finer than 2^-39 of the tensor's largest
// value: one token of 1e8 left 13 bits to values near 1.)
//
// The tensor core's float32 additions truncate: a sum of n of them is off by up to n 2^-23 and
// drifts towards zero (a loss of 16-bit rows of 65536 channels: 4e-5 off, of 1000 channels 4e-7; a
// rounding sum 1e-7).  So every stretch of the contraction is a sum of its own, small products first,
// and the epilogue warps add these sums in registers (rounding to nearest), under the products of the next.
// Float32 inputs: 64 at a time.  16-bit inputs: 1024 in logits, the same ones forward and backward (5e-7 at
// any length; 512 at a time: 2.5e-7 and 6 % of a step of 4096 x 32768 x 1024, whose G has no time left for
// it; 256 at a time: 1.3e-7, 20 % of the loss alone), and 256 for a loss alone of one tile per pair or less, where it
// costs nothing; 65536 in gradients (8e-6), which are rounded to 16 bits.
//
// Two CTAs on neighbouring SMs work as a pair (cta_group::2) on tiles of 256 x 256: each loads its own
// 128 rows of A and half of B, 32 KB per 64 of the contraction: 64 bytes per clock at the tensor core's
// rate, which is about what L2 delivers to an SM (128 x 256 tiles of one CTA: 96).  4096 x 32768 x 1024 in
// bfloat16: kLse 169 us (1.63 PFLOP/s, tensor pipe 95 % busy), kBack 358 us for twice the products
// (94 %), kGrad 220 us (70 %: its epilogue has a third more to do than the products leave time for).
// The float32 accumulators (256 columns of a CTA's tensor memory) are double-buffered, so that the
// epilogue of one tile runs under the products of the next.  Warp 0 issues the TMA loads, one thread of
// rank 0's warp 1 the products of the pair, warps 4..11 the epilogue (warp % 4 = the 32 rows it may
// read, (warp - 4) / 4 = the half of the columns).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include "f32x2.cuh"
#include "tma.cuh"
#include "umma.cuh"
#include "xent.h"

namespace msd {
namespace xent {

constexpr int kTileM = 256, kTileN = 256, kDepth = 64;  // of a pair
constexpr int kCtaM = 128, kCtaN = 128;                 // what each CTA loads: rows of A, columns of B
constexpr int kMmaThreads = 384;
constexpr int kABytes = kCtaM * kDepth * 2, kBBytes = kCtaN * kDepth * 2;
constexpr int kMaxPairs = 80;
constexpr int kTurn = 20;  // floats between the rows of a warp's transposing buffer (32 x 16): multiples of 16 bytes, 8 rows in 32 banks
constexpr int kRegsLaunch = 168, kRegsIssue = 40, kRegsEpilogue = 232;
static_assert(kRegsIssue * 128 + kRegsEpilogue * 256 <= kRegsLaunch * kMmaThreads, "a larger sum makes setmaxnreg.inc wait forever");

enum Use { kLse = 0, kGrad = 1, kBack = 2 };

// Blocks of 64 of the contraction whose products are added in the tensor core (powers of two).
constexpr int kSumSmall = 4, kSumStep = 16, kSumBack = 1024;
__host__ __device__ constexpr int stages_of(int pieces) { return pieces == 1 ? 6 : 2; }
__host__ __device__ constexpr size_t mma_smem_bytes(int pieces) {
    return 1024 + (size_t)stages_of(pieces) * pieces * (kABytes + kBBytes) + 2 * kTileN * sizeof(float) + 8 * 32 * kTurn * sizeof(float) + 256;
}

// One product: rows m of A, rows (or columns) n of B, contraction k.
struct Product {
    CUtensorMap a, b;
    int M, N, K;
    int tiles_m, tiles_n;
    int tile_n;                // columns of a tile: 256, or 192 or 128 where that fills the GPU better
    int splits, k_blocks;      // the contraction in blocks of 64, cut into `splits` ranges
    bool a_mn, b_mn;           // operand stored with m / n innermost instead of k
    bool parts;                // results go to `part`, to be joined, scaled and rounded later
    float *part;               // [split][M][ld] partial sums
    float *sum;                // [M][ld]: running float32 result over several pieces of the labels, or null
    int ld;                    // N rounded up to a multiple of 4
    bool add, last;            // add `sum` to the product; write `out` (else `sum`)
    bool vec;                  // rows of `out` are dense and take 16-byte stores throughout
    bool twos;                 // 16-bit rows that take 4-byte stores
    bool linear;               // t < V: row m lies at (row0 + m) sm
    void *out;                 // element (m, n) at (t / V) sn + (t % V) sm + n sc, t = row0 + m
    int64_t V, sn, sm, sc, row0;
};

// What the gradients are multiplied with: the product of two values on the device, or nothing.
struct Factor {
    const float *a, *b;
    __device__ __forceinline__ float value() const { return a ? *a * *b : 1.f; }
};

struct MmaParams {
    Product p[2];  // kLse, kGrad: [0]; kBack: [0] = dx, [1] = dW
    bool bf16;     // operand type: bfloat16, else float16
    int sum_blocks;  // one piece: one of these, else 1
    // kLse, kGrad
    const void *bias;
    int bias_type;
    const int64_t *target;
    int64_t ignore;
    int labels, label0;  // kGrad: this piece covers labels [label0, label0 + p[0].N)
    int group_m;         // rasterisation: this many row tiles pass before the next column tile
    float2 *part;        // kLse: [2 tiles_n][tokens] (maximum, sum of exp)
    float *zy;           // kLse: logit of the target
    Stats stats;  // kGrad: of the tokens
    const float *row_factor;  // kGrad: per token, or null: 1
    void *g;             // kGrad: [piece][tokens][g_width] 16-bit
    int64_t g_width, g_piece;
    float g_scale;       // power of two that G is held in
    float *columns;      // kGrad: [tokens / 32][g_width] sums of G over 32 tokens, or null
    Factor factor;       // kBack
    // kBack: pair i takes the items [first[0][i], first[0][i+1]) of product 0, then of product 1
    int first[2][kMaxPairs + 1];
    int *status;
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));  // off by 2^-22, relative
    return y;
}

__device__ __forceinline__ float load_float(const void *p, int type, int64_t i) {
    if (type == MSD_F32) return ((const float *)p)[i];
    if (type == MSD_BF16) return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
    return __half2float(((const __half *)p)[i]);
}

// Columns of a tile that are multiplied: the last tile only as many as it needs (both halves in
// multiples of 16).
__device__ __forceinline__ int columns_of(const Product &q, int n) { return min(q.tile_n, (q.N - n * q.tile_n + 31) / 32 * 32); }

struct Item {
    int which, m, n, k0, k1, split;
};

template <int USE>
struct Items {  // this pair's work, in order
    const MmaParams &p;
    int next, end, which;
    __device__ __forceinline__ explicit Items(const MmaParams &q) : p(q), which(0) {
        if (USE == kBack) {
            next = p.first[0][blockIdx.x >> 1], end = p.first[0][(blockIdx.x >> 1) + 1];
        } else {
            next = blockIdx.x >> 1, end = p.p[0].tiles_m * p.p[0].tiles_n;
        }
    }
    __device__ __forceinline__ bool get(Item &it) {
        if (USE == kBack) {
            if (next >= end) {
                if (which == 1) return false;
                which = 1;
                next = p.first[1][blockIdx.x >> 1], end = p.first[1][(blockIdx.x >> 1) + 1];
                if (next >= end) return false;
            }
            const Product &q = p.p[which];
            const int tile = next / q.splits;
            it.which = which, it.split = next % q.splits;
            it.m = tile / q.tiles_n, it.n = tile % q.tiles_n;
            it.k0 = (int)((int64_t)q.k_blocks * it.split / q.splits), it.k1 = (int)((int64_t)q.k_blocks * (it.split + 1) / q.splits);
            ++next;
            return true;
        }
        if (next >= end) return false;
        // column by column within groups of row tiles: W streams past once per group, x stays in L2
        const Product &q = p.p[0];
        const int per_group = p.group_m * q.tiles_n, group = next / per_group, in = next - group * per_group;
        const int rows = min(p.group_m, q.tiles_m - group * p.group_m);
        it.which = 0, it.split = 0, it.k0 = 0, it.k1 = q.k_blocks;
        it.m = group * p.group_m + in % rows, it.n = in / rows;
        next += gridDim.x >> 1;
        return true;
    }
};

// Results of P pieces: float32 for three, 16 bits for one.
template <int P>
__device__ __forceinline__ void store_one(void *out, bool bf16, int64_t i, float v) {
    if (P > 1) ((float *)out)[i] = v;
    else if (bf16) ((__nv_bfloat16 *)out)[i] = __float2bfloat16_rn(v);
    else ((__half *)out)[i] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t pack16(bool bf16, float a, float b) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// RUN: the contraction of a tile may be several sums, which are added in registers.
template <int USE, int P, bool RUN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMmaThreads, 1) xent_mma_kernel(const __grid_constant__ MmaParams p) {
    using namespace tma;
    static_assert(P == 1 || (P == 3 && RUN), "operands as they are, or in three pieces");
    constexpr bool WIDE = P > 1;
    const int F = WIDE ? 1 : RUN ? p.sum_blocks : 1 << 30;
    constexpr int S = stages_of(P);
    constexpr int kStage = P * (kABytes + kBBytes);
    extern __shared__ unsigned char xent_smem[];
    unsigned char *tiles = (unsigned char *)(((uintptr_t)xent_smem + 1023) & ~(uintptr_t)1023);
    float *bias_s = (float *)(tiles + S * kStage);  // [2][kTileN]
    float *turn_s = bias_s + 2 * kTileN;  // [8][32][kTurn]
    uint64_t *full = (uint64_t *)(turn_s + 8 * 32 * kTurn), *empty = full + S, *acc_full = empty + S, *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = (uint32_t *)(acc_empty + 2);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full + i, 1), mbar_init(acc_empty + i, 16);  // the epilogue warps of both CTAs
        *abort_flag = 0;
        fence_barrier_init();
    }
    const uint32_t rank = umma::cluster_rank();
    if (warp == 2) umma::tmem_alloc2(tmem_slot, 512);
    umma::fence_before_sync();
    umma::cluster_sync();  // both CTAs' barriers exist from here on
    umma::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // The epilogue warps keep 128 sums per thread.  kRegsIssue x 128 + kRegsEpilogue x 256 is
    // what the block was launched with (kRegsLaunch x 384; the launcher checks the compiled kernel).
    if (warp < 4) {
        if (RUN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        // The loops of both issuing warps run with all lanes (see umma::elect_one): with one lane in a
        // branch of its own the products of 64 took 1000 clocks to issue instead of the 512 they run.
        if (warp == 0) {
            Items<USE> items(p);
            Item it;
            int stage = 0;
            uint32_t phase = 0;
            while (items.get(it)) {
                const Product &q = p.p[it.which];
                const int n_cols = columns_of(q, it.n);
                const int m0 = it.m * kTileM + (int)rank * kCtaM, n0 = it.n * q.tile_n + (int)rank * (n_cols / 2);
                const bool a_mn = q.a_mn, b_mn = q.b_mn;
                for (int kb = it.k0; kb < it.k1; ++kb) {
                    wait_parity(empty + stage, phase ^ 1, abort_flag, p.status, 21);
                    __syncwarp();
                    unsigned char *a = tiles + stage * kStage, *b = a + P * kABytes;
                    // both CTAs' bytes are counted by rank 0, whose products wait for them
                    const uint32_t bar = umma::map_rank(smem_u32(full + stage), 0);
                    if (umma::elect_one()) {
                        if (rank == 0) mbar_arrive_expect_tx(full + stage, 2 * kStage);
#pragma unroll
                        for (int i = 0; i < P; ++i) {
                            if (a_mn) {
#pragma unroll
                                for (int h = 0; h < kCtaM / 64; ++h)
                                    umma::tensor_g2s_3d_pair(a + i * kABytes + h * 8192, &q.a, m0 + h * 64, kb * kDepth, i, bar);
                            } else {
                                umma::tensor_g2s_3d_pair(a + i * kABytes, &q.a, kb * kDepth, m0, i, bar);
                            }
                            if (b_mn) {
#pragma unroll
                                for (int h = 0; h < kCtaN / 64; ++h)
                                    umma::tensor_g2s_3d_pair(b + i * kBBytes + h * 8192, &q.b, n0 + h * 64, kb * kDepth, i, bar);
                            } else {
                                umma::tensor_g2s_3d_pair(b + i * kBBytes, &q.b, kb * kDepth, n0, i, bar);
                            }
                        }
                    }
                    __syncwarp();
                    if (++stage == S) stage = 0, phase ^= 1;
                }
            }
        }
        if (warp == 1 && rank == 0) {
            Items<USE> items(p);
            Item it;
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            // descriptors differ in their start address only (units of 16 bytes)
            const uint64_t d0 = umma::smem_desc_sw128(smem_u32(tiles), 8192, 1024);
            const uint32_t lo0 = (uint32_t)d0, hi = (uint32_t)(d0 >> 32);
            while (items.get(it)) {
                const Product &q = p.p[it.which];
                const int n_cols = columns_of(q, it.n), K = q.K;
                const uint32_t idesc = umma::idesc_f16(p.bf16, kTileM, n_cols, q.a_mn, q.b_mn);
                // K-major: 8-row atoms follow at 1024 bytes, 16 k = 32 bytes.  MN-major: blocks of 64 follow at
                // 8192 bytes, 8 k at 1024, so 16 k = 2048 bytes.
                const uint32_t a_step = q.a_mn ? 2048 / 16 : 32 / 16, b_step = q.b_mn ? 2048 / 16 : 32 / 16;
                for (int kb = it.k0; kb < it.k1; ++kb) {
                    const bool first = ((kb - it.k0) & (F - 1)) == 0;
                    if (first) {
                        wait_parity(acc_empty + acc, acc_phase ^ 1, abort_flag, p.status, 22);
                        __syncwarp();
                        umma::fence_after_sync();
                    }
                    const uint32_t d = tmem + acc * kTileN;
                    wait_parity(full + stage, phase, abort_flag, p.status, 23);
                    __syncwarp();
                    umma::fence_after_sync();
                    const uint32_t a = lo0 + (uint32_t)(stage * kStage) / 16, b = a + P * kABytes / 16;
                    const int steps = min(kDepth / 16, (K - kb * kDepth + 15) / 16);
                    const bool sum_done = ((kb - it.k0) & (F - 1)) == F - 1 || kb + 1 == it.k1;
                    if (umma::elect_one()) {
                        // pieces whose orders add up to 2, then 1, then 0: the small products first
#pragma unroll
                        for (int order = P - 1; order >= 0; --order)
#pragma unroll
                            for (int ks = 0; ks < kDepth / 16; ++ks)
                                if (ks < steps)
#pragma unroll
                                    for (int i = 0; i <= order; ++i)
                                        umma::mma_f16_pair(d, umma::desc_words(a + i * (kABytes / 16) + ks * a_step, hi),
                                                           umma::desc_words(b + (order - i) * (kBBytes / 16) + ks * b_step, hi), idesc,
                                                           order < P - 1 || ks > 0 || i > 0 || !first);
                        umma::commit_pair(empty + stage);
                        if (sum_done) umma::commit_pair(acc_full + acc);
                    }
                    __syncwarp();
                    if (++stage == S) stage = 0, phase ^= 1;
                    if (sum_done && ++acc == 2) acc = 0, acc_phase ^= 1;
                }
            }
        }
        __syncwarp();
    } else {
        if (RUN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue));
        const int half = (warp - 4) >> 2, quad = warp & 3;
        Items<USE> items(p);
        Item it;
        int acc = 0;
        uint32_t acc_phase = 0;
        int parity = 0, biases_of = -1;
        Pair sums[RUN ? kTileN / 4 : 1];  // of the contraction so far
        while (items.get(it)) {
            const Product &q = p.p[it.which];
            const int row = it.m * kTileM + (int)rank * kCtaM + quad * 32 + lane;  // token (kBack, dW: label)
            const int width = q.tile_n / 2, col0 = it.n * q.tile_n + half * width;  // this half's columns
            const int cols = min(width, q.N - col0);                                // may be 0 or less
            // read while the products run
            const bool in = row < q.M;
            int64_t y = p.ignore;
            float lse = 0.f, rest = 0.f, upstream = 1.f;
            if (USE != kBack && in) y = p.target[row];
            if (USE == kGrad && in) {
                p.stats.read(row, lse, rest);
                if (p.row_factor) upstream = p.row_factor[row];
            }
            if (USE != kBack && it.n != biases_of) {
                // this half's biases; labels past the end count as -infinity
                biases_of = it.n, parity ^= 1;
                const int i = threadIdx.x - 128 - half * 128, o = p.label0 + col0 + i;
                bias_s[parity * kTileN + half * (kTileN / 2) + i] =
                    i < cols && o < p.labels ? (p.bias ? load_float(p.bias, p.bias_type, o) : 0.f) : -CUDART_INF_F;
                named_barrier(1 + half, 128);
            }
            const float *bias_h = bias_s + parity * kTileN + half * (kTileN / 2);
            uint32_t t0 = 0;  // the tile in tensor memory, unless its sums are in registers
            if constexpr (RUN) {
                // They leave the tensor memory to the next products at once: with the arithmetic below in
                // between, the products of the next tile would wait for it.
#pragma unroll
                for (int j = 0; j < kTileN / 4; ++j) sums[j] = pair(0.f, 0.f);
                for (int kb = it.k0; kb < it.k1; kb += F) {
                    wait_parity(acc_full + acc, acc_phase, abort_flag, p.status, 24);
                    __syncwarp();
                    umma::fence_after_sync();
                    const uint32_t t = tmem + acc * kTileN + half * width + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                    for (int c = 0; c < kTileN / 2; c += 32) {
                        if (c >= cols) continue;
                        uint32_t r[32];
                        umma::tmem_ld32_issue(t + c, r);
                        umma::tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) sums[c / 2 + j] = add2(sums[c / 2 + j], pair(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])));
                    }
                    umma::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) umma::arrive_at(umma::map_rank(smem_u32(acc_empty + acc), 0));
                    if (++acc == 2) acc = 0, acc_phase ^= 1;
                }
            } else {
                wait_parity(acc_full + acc, acc_phase, abort_flag, p.status, 24);
                __syncwarp();
                umma::fence_after_sync();
                t0 = tmem + acc * kTileN + half * width + ((uint32_t)(quad * 32) << 16);
            }
            // Columns [c, c + 32) of this half.  From tensor memory in a loop of 32 columns: straight-line code for
            // all of them runs once per tile and waits for its instructions (dx of 2 million voxels: 1150 us
            // against 690).
            const auto take = [&](int c, Pair (&x)[16]) {
                if constexpr (RUN) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = sums[c / 2 + j];
                } else {
                    uint32_t r[32];
                    __syncwarp();
                    umma::tmem_ld32_issue(t0 + c, r);
                    umma::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = pair(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                }
            };
            if (USE == kLse) {
                float top = -CUDART_INF_F, sum = 0.f;
                const bool live = in;
                const int hit = live && y >= col0 && y < col0 + cols ? (int)(y - col0) : -1;
#pragma unroll(RUN ? 4 : 1)
                for (int c = 0; c < kTileN / 2; c += 32) {
                    if (c >= cols) continue;
                    Pair x[16];
                    take(c, x);
                    float z[32], m = -CUDART_INF_F;
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const ulonglong2 b4 = *reinterpret_cast<const ulonglong2 *>(bias_h + c + 2 * j);
                        unpair(add2(x[j], b4.x), z[2 * j], z[2 * j + 1]);
                        unpair(add2(x[j + 1], b4.y), z[2 * j + 2], z[2 * j + 3]);
                    }
                    if (c + 32 > cols) {  // columns that no product wrote
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c + j >= cols) z[j] = -CUDART_INF_F;
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) m = fmaxf(m, z[j]);
                    if (__any_sync(0xffffffffu, hit >= c && hit < c + 32)) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (hit == c + j) p.zy[row] = z[j];
                    }
                    const float up = fmaxf(top, m);
                    const float base = up == -CUDART_INF_F ? 0.f : up;
                    Pair s[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                    const Pair off = pair(-base, -base), scale = pair(kLog2e, kLog2e);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float e0, e1;
                        unpair(mul2(add2(pair(z[2 * j], z[2 * j + 1]), off), scale), e0, e1);
                        s[j & 1] = add2(s[j & 1], pair(exp2_fast(e0), exp2_fast(e1)));  // a NaN logit makes the sum NaN
                    }
                    float s0, s1;
                    unpair(add2(s[0], s[1]), s0, s1);
                    sum = sum * exp2_fast((top - base) * kLog2e) + (s0 + s1);
                    top = up;
                }
                if (live && !*abort_flag) p.part[(int64_t)(2 * it.n + half) * q.M + row] = make_float2(top, sum);
            } else if (USE == kGrad) {
                const bool live = in, counts = live && y != p.ignore;
                float g = counts ? upstream * p.g_scale : 0.f;
                if (counts && (y < 0 || y >= p.labels)) g = CUDART_NAN_F;
                const int hit = counts && y >= p.label0 + col0 && y < p.label0 + col0 + cols ? (int)(y - p.label0 - col0) : -1;
                const bool all_count = __all_sync(0xffffffffu, counts);
                const Pair off = pair(-lse, -lse), off_rest = pair(rest * -kLog2e, rest * -kLog2e), scale = pair(kLog2e, kLog2e), factor = pair(g, g);
                const int stored = (int)min((int64_t)width, p.g_width - col0);
                const bool ok = !*abort_flag;
                float *turn = turn_s + (warp - 4) * 32 * kTurn;
#pragma unroll(RUN ? 4 : 1)
                for (int c = 0; c < kTileN / 2; c += 32) {
                    if (c >= stored) continue;
                    Pair x[16];
                    take(c, x);
                    float v[32];  // log2 p
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const ulonglong2 b4 = *reinterpret_cast<const ulonglong2 *>(bias_h + c + 2 * j);
                        unpair(fma2(add2(add2(x[j], b4.x), off), scale, off_rest), v[2 * j], v[2 * j + 1]);
                        unpair(fma2(add2(add2(x[j + 1], b4.y), off), scale, off_rest), v[2 * j + 2], v[2 * j + 3]);
                    }
                    float d = 0.f;  // p - 1 of the target: exact where p is close to 1
                    const bool any = __any_sync(0xffffffffu, hit >= c && hit < c + 32);
                    if (any) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) d = hit == c + j ? v[j] : d;
                        d = expm1f(d * kLn2);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = exp2_fast(v[j]);
                    if (any) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = hit == c + j ? d : v[j];
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) unpair(mul2(pair(v[2 * j], v[2 * j + 1]), factor), v[2 * j], v[2 * j + 1]);
                    if (c + 32 > cols || !all_count) {  // past the last label, and ignored tokens: exact zeros whatever the logits hold
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = counts && c + j < cols ? v[j] : 0.f;
                    }
                    // A lane has 64 bytes of its row.  Stored like that, every store touches 32 rows (292 us for
                    // 4096 x 32768 x 1024, 207 without the stores); turned in shared memory, it writes whole
                    // 64-byte pieces of 8 rows (229).
#pragma unroll
                    for (int piece = 0; piece < P; ++piece) {
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            if (P == 1) {
                                w[j] = pack16(p.bf16, v[2 * j], v[2 * j + 1]);
                            } else {
                                float v0 = v[2 * j], v1 = v[2 * j + 1];
#pragma unroll
                                for (int i = 0; i < piece; ++i) {
                                    const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
                                    v0 -= __low2float(h), v1 -= __high2float(h);
                                }
                                w[j] = pack16(true, v0, v1);
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<uint4 *>(turn + lane * kTurn + 4 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                        __syncwarp();
                        const int j = lane & 3;
                        uint16_t *dst = (uint16_t *)p.g + piece * p.g_piece + (int64_t)(row - lane) * p.g_width + col0 + c + 8 * j;
#pragma unroll
                        for (int i = lane >> 2; i < 32; i += 8)
                            if (ok && row - lane + i < q.M && c + 8 * j < stored)
                                *reinterpret_cast<uint4 *>(dst + i * p.g_width) = *reinterpret_cast<const uint4 *>(turn + i * kTurn + 4 * j);
                    }
                    if (p.columns) {
                        // reduce-scatter over the warp's 32 tokens: lane l ends up with column l
#pragma unroll
                        for (int w = 16; w > 0; w >>= 1) {
                            const bool up = lane & w;
#pragma unroll
                            for (int i = 0; i < w; ++i) {
                                const float mine = up ? v[i + w] : v[i], give = up ? v[i] : v[i + w];
                                v[i] = mine + __shfl_xor_sync(0xffffffffu, give, w);
                            }
                        }
                        if (ok && row - lane < q.M && c + lane < stored) p.columns[(int64_t)(row >> 5) * p.g_width + col0 + c + lane] = v[0];
                    }
                }
            } else {
                const bool ok = !*abort_flag, live = row < q.M && ok;
                const float f = p.factor.value() / p.g_scale;
                const bool split = q.parts, done = !split && q.last;
                float *run = split ? q.part + ((int64_t)it.split * q.M + row) * q.ld : q.sum + (int64_t)row * q.ld;
                const bool add = !split && q.add;
                const int64_t at = q.linear ? (q.row0 + row) * q.sm : ((q.row0 + row) / q.V) * q.sn + ((q.row0 + row) % q.V) * q.sm;
                float *turn = turn_s + (warp - 4) * 32 * kTurn;
#pragma unroll(RUN ? 4 : 1)
                for (int c = 0; c < kTileN / 2; c += 32) {
                    if (c >= cols) continue;
                    Pair x[16];
                    take(c, x);
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 16; ++j) unpair(x[j], v[2 * j], v[2 * j + 1]);
                    const int col = col0 + c;
                    if (add && live) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            if (c + j < cols) {
                                const float4 o = *reinterpret_cast<const float4 *>(run + col + j);
                                v[j] += o.x, v[j + 1] += o.y, v[j + 2] += o.z, v[j + 3] += o.w;
                            }
                    }
                    if (!done) {
                        if (live) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4)
                                if (c + j < cols) *reinterpret_cast<float4 *>(run + col + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        }
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] *= f;
                    if (q.vec) {  // 16-byte pieces, 64 bytes of a row together: turned as in kGrad
#pragma unroll
                        for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if (WIDE) {
                                    const float *f = v + 16 * h + 4 * j;
                                    *reinterpret_cast<float4 *>(turn + lane * kTurn + 4 * j) = make_float4(f[0], f[1], f[2], f[3]);
                                } else {
                                    const float *f = v + 8 * j;
                                    *reinterpret_cast<uint4 *>(turn + lane * kTurn + 4 * j) =
                                        make_uint4(pack16(p.bf16, f[0], f[1]), pack16(p.bf16, f[2], f[3]), pack16(p.bf16, f[4], f[5]), pack16(p.bf16, f[6], f[7]));
                                }
                            }
                            __syncwarp();
                            const int j = lane & 3, piece = WIDE ? 16 * h + 4 * j : 8 * j;  // first of the lane's columns
#pragma unroll
                            for (int i = lane >> 2; i < 32; i += 8) {
                                const int64_t there = __shfl_sync(0xffffffffu, at, i) + col + piece;
                                if (ok && row - lane + i < q.M && c + piece < cols)
                                    *reinterpret_cast<uint4 *>((char *)q.out + there * (WIDE ? 4 : 2)) = *reinterpret_cast<const uint4 *>(turn + i * kTurn + 4 * j);
                            }
                        }
                    } else if (q.sc != 1) {  // neighbouring tokens lie side by side: each column is a dense store of the warp
                        if (live) {
                            int64_t o = at + (int64_t)col * q.sc;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                if (c + j < cols) store_one<P>(q.out, p.bf16, o, v[j]);
                                o += q.sc;
                            }
                        }
                    } else {  // dense rows without a common alignment: 16 columns of some rows at a time
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4 *>(turn + lane * kTurn + j) = make_float4(v[h + j], v[h + j + 1], v[h + j + 2], v[h + j + 3]);
                            __syncwarp();
                            const int left = min(16, cols - c - h), rows = ok ? min(32, q.M - (row - lane)) : 0;
                            if (P == 1 && q.twos && q.linear) {  // 4 rows x 8 pairs
                                const int j = 2 * (lane & 7), i0 = lane >> 3;
                                uint16_t *to = (uint16_t *)q.out + (q.row0 + row - lane + i0) * q.sm + col + h + j;
                                const float *from = turn + i0 * kTurn + j;
                                const bool in = j < left;
#pragma unroll
                                for (int i = 0; i < 32; i += 4, to += 4 * q.sm, from += 4 * kTurn) {
                                    const float2 f = *reinterpret_cast<const float2 *>(from);
                                    if (in && i0 + i < rows) *reinterpret_cast<uint32_t *>(to) = pack16(p.bf16, f.x, f.y);
                                }
                            } else {  // 2 rows x 16
                                const int j = lane & 15;
#pragma unroll 4
                                for (int i = lane >> 4; i < 32; i += 2) {
                                    const int64_t there = __shfl_sync(0xffffffffu, at, i) + col + h;
                                    if (i < rows && j < left) store_one<P>(q.out, p.bf16, there + j, turn[i * kTurn + j]);
                                }
                            }
                        }
                    }
                }
            }
            if constexpr (!RUN) {
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) umma::arrive_at(umma::map_rank(smem_u32(acc_empty + acc), 0));
                if (++acc == 2) acc = 0, acc_phase ^= 1;
            }
        }
    }
    umma::fence_before_sync();
    umma::cluster_sync();  // neither CTA leaves while the other may still arrive at its barriers
    if (warp == 2) umma::tmem_dealloc2(tmem, 512);
}

}  // namespace xent
}  // namespace msd
