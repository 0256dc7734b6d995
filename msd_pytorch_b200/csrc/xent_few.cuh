// Linear layer with softmax cross entropy for a handful of tokens (scoring a token against a large
// vocabulary): a matrix-vector product, bound by reading W once.
//
// x is held in shared memory as float32.  A warp takes four rows of W at a time (16 bytes per lane
// and row, so that x's values are read from shared memory once per four rows), adds the products in
// float32, joins its lanes' sums by shuffles and carries a running (maximum, sum of exp) per token
// over its rows.  The block's warps are joined at the end: one pair per block and token.  Whole calls, W read from
// HBM, here and as tiles of the tensor-core kernel: 50000 rows of 2048 bfloat16 for 1, 2 and 4 tokens 49, 59 and 68
// us against 82, 86 and 78; 5003 rows of 1024 16, 16 and 21 against 25; 5 tokens and more: as tiles.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <string.h>
#include <atomic>
#include "xent.h"

namespace msd {
namespace xent {

constexpr int kFewTokens = 4;
constexpr int kFewRows = 4, kFewWarps = 16;
constexpr int kFewBlocks = 592;  // at most; two per SM
constexpr int64_t kFewChannels = 8192;  // x takes 128 KB of shared memory

struct FewParams {
    Features x;
    const void *weight, *bias;
    const int64_t *target;
    int64_t ignore, O;
    int T, C4;  // tokens; channels as held in shared memory
    bool vec;   // rows of W take 16-byte loads
    float2 *part;  // [block][T]
    float *zy;
};

inline bool few_supported(const Problem &p) { return p.x.tokens() <= kFewTokens && p.x.C <= kFewChannels; }

template <typename T>
__device__ __forceinline__ float few_float(T v);
template <>
__device__ __forceinline__ float few_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float few_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float few_float<__half>(__half v) { return __half2float(v); }

template <typename T, int N, bool VEC>
__global__ void __launch_bounds__(32 * kFewWarps) few_kernel(const FewParams p) {
    extern __shared__ __align__(16) float few_x[];  // [N][C4], zeros past the last channel and for ignored tokens
    __shared__ float2 red[kFewWarps][N];
    const int C = (int)p.x.C, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int t = 0; t < N; ++t) {
        const bool in = t < p.T && p.target[t] != p.ignore;
        const T *row = (const T *)p.x.p + (t / p.x.V) * p.x.sn + (t % p.x.V) * p.x.sv;
        for (int c = threadIdx.x; c < p.C4; c += 32 * kFewWarps) few_x[t * p.C4 + c] = in && c < C ? few_float<T>(row[c * p.x.sc]) : 0.f;
    }
    __syncthreads();
    int64_t y[N];
    float top[N], sum[N];
#pragma unroll
    for (int t = 0; t < N; ++t) {
        y[t] = t < p.T ? p.target[t] : -1;
        top[t] = -CUDART_INF_F, sum[t] = 0.f;
    }
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
    const T *w = (const T *)p.weight;
    for (int64_t o0 = ((int64_t)blockIdx.x * kFewWarps + warp) * kFewRows; o0 < p.O; o0 += (int64_t)gridDim.x * kFewWarps * kFewRows) {
        float acc[kFewRows][N];
        const T *row[kFewRows];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            row[r] = w + min(o0 + r, p.O - 1) * C;
#pragma unroll
            for (int t = 0; t < N; ++t) acc[r][t] = 0.f;
        }
#pragma unroll 2
        for (int c = lane * E; c < C; c += 32 * E) {
            T v[kFewRows][E];
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                if (VEC) {
                    const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(row[r] + c));
                    memcpy(v[r], &u, sizeof(v[r]));
                } else {
                    v[r][0] = row[r][c];
                }
            }
#pragma unroll
            for (int t = 0; t < N; ++t) {
                float xv[E];
                if (VEC) {
#pragma unroll
                    for (int k = 0; k < E; k += 4) *reinterpret_cast<float4 *>(xv + k) = *reinterpret_cast<const float4 *>(few_x + t * p.C4 + c + k);
                } else {
                    xv[0] = few_x[t * p.C4 + c];
                }
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
#pragma unroll
                    for (int k = 0; k < E; ++k) acc[r][t] = fmaf(few_float<T>(v[r][k]), xv[k], acc[r][t]);
            }
        }
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            if (o0 + r >= p.O) continue;
            const float b = p.bias ? few_float<T>(((const T *)p.bias)[o0 + r]) : 0.f;
#pragma unroll
            for (int t = 0; t < N; ++t) {
                float z = acc[r][t];
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) z += __shfl_xor_sync(0xffffffffu, z, off);
                z += b;
                if (lane == 0 && t < p.T && o0 + r == y[t]) p.zy[t] = z;
                const float up = fmaxf(top[t], z), base = up == -CUDART_INF_F ? 0.f : up;
                sum[t] = sum[t] * exp2f((top[t] - base) * kLog2e) + exp2f((z - base) * kLog2e);  // a NaN logit makes the sum NaN
                top[t] = up;
            }
        }
    }
    if (lane == 0)
#pragma unroll
        for (int t = 0; t < N; ++t) red[warp][t] = make_float2(top[t], sum[t]);
    __syncthreads();
    if (threadIdx.x < p.T) {
        float m = -CUDART_INF_F, s = 0.f;
        for (int i = 0; i < kFewWarps; ++i) {
            const float2 v = red[i][threadIdx.x];
            const float up = fmaxf(m, v.x), base = up == -CUDART_INF_F ? 0.f : up;
            s = s * exp2f((m - base) * kLog2e) + v.y * exp2f((v.x - base) * kLog2e);
            m = up;
        }
        p.part[(int64_t)blockIdx.x * p.T + threadIdx.x] = make_float2(m, s);
    }
}

// Joins the blocks and reduces the losses: one warp per token.
__global__ void __launch_bounds__(32 * kFewTokens) few_finish_kernel(const float2 *part, const float *zy, const int64_t *target, int64_t ignore, int T_, int64_t O,
                                                                    int blocks, int reduction, float *loss, const Stats saved) {
    __shared__ float losses[kFewTokens];
    const int t = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (t < T_) {
        float m = -CUDART_INF_F, s = 0.f;
        const auto join = [&](float m2, float s2) {
            const float up = fmaxf(m, m2), base = up == -CUDART_INF_F ? 0.f : up;
            s = s * exp2f((m - base) * kLog2e) + s2 * exp2f((m2 - base) * kLog2e);
            m = up;
        };
#pragma unroll 4
        for (int i = lane; i < blocks; i += 32) {
            const float2 v = part[(int64_t)i * T_ + t];
            join(v.x, v.y);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off);
            join(m2, s2);
        }
        if (lane == 0) {
            const float log_s = logf(s);
            const int64_t y = target[t];
            losses[t] = y == ignore ? 0.f : y >= 0 && y < O ? (m - zy[t]) + log_s : CUDART_NAN_F;  // NaN: a target that names no label
            if (saved.lse) saved.write(t, m, log_s);
            if (reduction == MSD_REDUCE_NONE) loss[t] = losses[t];
        }
    }
    __syncthreads();
    if (threadIdx.x) return;
    double total = 0;
    int count = 0;
    for (int i = 0; i < T_; ++i) total += losses[i], count += target[i] != ignore;
    if (reduction == MSD_REDUCE_MEAN) loss[0] = (float)(total / (double)count);
    if (reduction == MSD_REDUCE_SUM) loss[0] = (float)total;
    if (saved.lse) *saved.factor = reduction == MSD_REDUCE_MEAN ? (count ? (float)(1.0 / (double)count) : 0.f) : 1.f;
}

template <typename T, int N>
static int launch_few_tokens(const FewParams &p, int blocks, cudaStream_t s) {
    auto kern = p.vec ? few_kernel<T, N, true> : few_kernel<T, N, false>;
    const size_t smem = (size_t)N * p.C4 * sizeof(float);
    // the most that any call takes, once: the limit is shared by all threads of the process
    static std::atomic<uint64_t> ready[2];
    int device = 0;
    MSD_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 64 || !(ready[p.vec].load() >> device & 1)) {
        MSD_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(N * kFewChannels * sizeof(float))));
        if (device < 64) ready[p.vec].fetch_or(1ull << device);
    }
    kern<<<blocks, 32 * kFewWarps, smem, s>>>(p);
    MSD_CUDA_TRY(cudaGetLastError());
    return MSD_OK;
}
template <typename T>
static int launch_few(const FewParams &p, int blocks, cudaStream_t s) {
    return p.T == 1 ? launch_few_tokens<T, 1>(p, blocks, s) : p.T == 2 ? launch_few_tokens<T, 2>(p, blocks, s) : launch_few_tokens<T, 4>(p, blocks, s);
}

}  // namespace xent
}  // namespace msd
