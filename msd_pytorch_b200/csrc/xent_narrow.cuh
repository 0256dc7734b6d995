// Linear layer with softmax cross entropy for few labels (at most 16) and voxels that lie side by
// side in memory: the segmentation network's own case, bound by HBM.
//
// The logits of a voxel need all its channels before any of its gradients can be formed, and dx, dW
// need the channels again.  A block therefore holds a tile of 64 voxels with ALL channels in
// shared memory (29 KB for 101 float32 channels; up to four tiles in flight with cp.async):
// x is read once and dx written once.  Per tile:
//   1  a warp takes 8 voxels, its four groups of lanes a quarter of the channels each: partial
//      logits; a shuffle reduce-scatter leaves every lane the logits of a quarter of the labels;
//      softmax, loss, G -> shared memory.  Rows are 72 elements apart, so that the groups' rows lie
//      in different banks.
//   2  a half warp takes every 16th channel, a lane four voxels: dx, stored at once, and the sums
//      over the lane's voxels of G x.  With up to 128 channels and 4 labels these sums stay in
//      registers from tile to tile; otherwise a shuffle reduce-scatter adds 16 (label, channel) sums at
//      a time into sums in shared memory.
// Two blocks per SM: one's loads and arithmetic run
// under the other's barriers.  Two 1024 x 1024 images, 101 channels, 4 labels: 405 to 420 us, 4.1 TB/s,
// bound by latency (issue slots 55 % busy; 122 registers leave 16 warps per SM); one block of 16
// warps with tiles of 128 voxels: 472.
//
// float32 products on the CUDA cores, two per instruction (fma.rn.f32x2).  The instruction stream is
// what had to shrink: a first version issued 26000 warp instructions per 128 voxels (101 channels, 4
// labels; now 15300) and took 523 us with the issue slots 73 % busy.  Sums over the blocks run in a fixed
// order in float64.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include "f32x2.cuh"
#include "xent.h"

namespace msd {
namespace xent {

constexpr int kNarrowLabels = 16;
constexpr int kVoxels = 64;        // per tile
constexpr int kRow = kVoxels + 8;  // elements between the rows of a tile in shared memory
constexpr int kWarps = 8;          // of a block
constexpr int kSlots = 2 * kWarps;    // half warps: each takes every 16th channel in part 2
constexpr int kRegisterChannels = 8;  // channels of a half warp whose sums of dW can stay in registers

struct NarrowParams {
    const void *x;
    int64_t N, V, sn, sc;
    int C, O;
    const void *weight, *bias;
    const int64_t *target;
    int64_t ignore;
    // gradients
    void *dx;
    int64_t dn, dc;
    bool want_dx;
    const float *grad_loss;  // null: 1
    bool per_token;          // grad_loss per token
    const float *mean_factor;  // factor of a mean (what forward left), or null
    const int64_t *counted;    // instead: the number of tokens that count,
    int count_here;            // or, above 0, every block counts the targets itself
    bool mean;
    float *part;             // [block][16 C + 16]: sums of dW, then db
    // loss
    float *losses;           // per token, or null
    double *block_sum;
    int64_t *block_count;
    int64_t tiles_per_image, tiles;
    int step_images, step_tiles;  // the number of blocks, in images and tiles
    int stages;
};

template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T as_type(float v);
template <>
__device__ __forceinline__ float as_type<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half as_type<__half>(float v) { return __float2half_rn(v); }

template <typename T>
struct alignas(4 * sizeof(T)) Quad {
    T v[4];
};

// Voxel j of lane l of a half warp, in part 2: four neighbours where rows are aligned for vector
// accesses, else 16 apart (scalar accesses of a half warp then cover whole sectors).
template <bool ALIGNED>
__device__ __forceinline__ int voxel_of(int lane, int j) { return ALIGNED ? 4 * lane + j : lane + 16 * j; }

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_voxels(const T *row, int lane, float (&v)[4]) {
    if (ALIGNED) {
        const Quad<T> q = *reinterpret_cast<const Quad<T> *>(row + 4 * lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = as_float<T>(q.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = as_float<T>(row[lane + 16 * j]);
    }
}

template <int OP>
__device__ __forceinline__ void load_weights(const float *ws, float (&w)[OP]) {
#pragma unroll
    for (int o = 0; o < OP; o += 4) {
        const float4 q = *reinterpret_cast<const float4 *>(ws + o);
        w[o] = q.x, w[o + 1] = q.y, w[o + 2] = q.z, w[o + 3] = q.w;
    }
}

__device__ __forceinline__ float exp2_narrow(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- the loss alone: a stream over x ---------------------------------------------------------------
// A lane keeps the logits of its voxels (four neighbours; two from 13 labels on) in registers and passes
// over all channels, eight loads in flight; the weights lie in shared memory, each twice, so that one
// 16-byte load brings two labels' packed operands.  Bound by latency and shared memory: 49 us for
// 792288 voxels, 51 channels and 11 labels (26 at the HBM rate; two voxels per lane: 52; the next
// loads ahead of the arithmetic: 50; as the gradient kernel's first part, with 2.4 times the
// instructions: 74).
__host__ __device__ constexpr int loss_voxels(int OP) { return OP > 12 ? 2 : 4; }
constexpr int kLossDepth = 8;

template <typename T, int K>
struct alignas(K * sizeof(T)) Vec {
    T v[K];
};

template <typename T, int OP, bool ALIGNED>
__global__ void __launch_bounds__(32 * kWarps, OP == 8 || OP == 12 ? 2 : 3) narrow_loss_kernel(const __grid_constant__ NarrowParams p) {
    constexpr int K = loss_voxels(OP), THREADS = 32 * kWarps;
    extern __shared__ __align__(16) float narrow_smem[];
    Pair *ws = reinterpret_cast<Pair *>(narrow_smem);  // [C][OP]
    float *bs = narrow_smem + 2 * p.C * OP;            // [OP]
    for (int i = threadIdx.x; i < p.C * OP; i += THREADS) {
        const int c = i / OP, o = i % OP;
        const float w = o < p.O ? as_float<T>(((const T *)p.weight)[(int64_t)o * p.C + c]) : 0.f;
        ws[i] = pair(w, w);
    }
    if (threadIdx.x < OP) bs[threadIdx.x] = threadIdx.x < p.O ? (p.bias ? as_float<T>(((const T *)p.bias)[threadIdx.x]) : 0.f) : -CUDART_INF_F;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double total = 0;
    int count = 0;
    const int per_image = (int)((p.V + 32 * K - 1) / (32 * K));
    const int64_t tiles = p.N * per_image;
    for (int64_t tile = blockIdx.x * (int64_t)kWarps + warp; tile < tiles; tile += (int64_t)gridDim.x * kWarps) {
        const int n = (int)((uint32_t)tile / (uint32_t)per_image);
        const int64_t v0 = (int64_t)((uint32_t)tile % (uint32_t)per_image) * (32 * K);
        const bool full = v0 + 32 * K <= p.V;
        int64_t y[K];  // read under the channels
        bool in[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int64_t v = v0 + (ALIGNED ? K * lane + j : lane + 32 * j);
            in[j] = v < p.V;
            y[j] = in[j] ? p.target[n * p.V + v] : p.ignore;
        }
        const T *x = (const T *)p.x + n * p.sn + v0 + (ALIGNED ? K * lane : lane);
        Pair z2[K / 2][OP];
#pragma unroll
        for (int j = 0; j < K / 2; ++j)
#pragma unroll
            for (int o = 0; o < OP; ++o) z2[j][o] = pair(0.f, 0.f);
        const Pair *w = ws;
        const auto load = [&](const T *at, float (&v)[K]) {
            if (ALIGNED && full) {
                const Vec<T, K> q = *reinterpret_cast<const Vec<T, K> *>(at);
#pragma unroll
                for (int j = 0; j < K; ++j) v[j] = as_float<T>(q.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < K; ++j) v[j] = in[j] ? as_float<T>(at[ALIGNED ? j : 32 * j]) : 0.f;
            }
        };
        const auto add = [&](const float (&v)[K]) {
#pragma unroll
            for (int o = 0; o < OP; o += 2) {
                const ulonglong2 ww = *reinterpret_cast<const ulonglong2 *>(w + o);
#pragma unroll
                for (int j = 0; j < K / 2; ++j) {
                    const Pair vv = pair(v[2 * j], v[2 * j + 1]);
                    z2[j][o] = fma2(ww.x, vv, z2[j][o]), z2[j][o + 1] = fma2(ww.y, vv, z2[j][o + 1]);
                }
            }
            w += OP;
        };
        int c = 0;
        for (; c + kLossDepth <= p.C; c += kLossDepth) {
            float v[kLossDepth][K];
#pragma unroll
            for (int i = 0; i < kLossDepth; ++i, x += p.sc) load(x, v[i]);
#pragma unroll
            for (int i = 0; i < kLossDepth; ++i) add(v[i]);
        }
        for (; c < p.C; ++c, x += p.sc) {
            float v[K];
            load(x, v);
            add(v);
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            float z[OP], top = -CUDART_INF_F;
#pragma unroll
            for (int o = 0; o < OP; ++o) {
                float a, b;
                unpair(z2[j / 2][o], a, b);
                z[o] = (j & 1 ? b : a) + bs[o];
                top = fmaxf(top, z[o]);
            }
            const float base = top == -CUDART_INF_F ? 0.f : top;
            const int hit = y[j] >= 0 && y[j] < p.O ? (int)y[j] : -1;
            float s = 0.f, chosen = 0.f;
#pragma unroll
            for (int o = 0; o < OP; ++o) {
                s += exp2_narrow((z[o] - base) * kLog2e);  // NaN logits: a NaN sum
                if (o == hit) chosen = z[o];
            }
            float loss = 0.f;
            if (y[j] != p.ignore) {
                loss = hit >= 0 ? (base - chosen) + logf(s) : CUDART_NAN_F;  // no label left: infinity - infinity
                ++count;
            }
            if (p.losses && in[j]) p.losses[n * p.V + v0 + (ALIGNED ? K * lane + j : lane + 32 * j)] = loss;
            total += loss;
        }
    }
    __shared__ double rsum[kWarps];
    __shared__ int64_t rcount[kWarps];
    int64_t counted = count;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        total += __shfl_down_sync(0xffffffffu, total, off);
        counted += __shfl_down_sync(0xffffffffu, counted, off);
    }
    if (lane == 0) rsum[warp] = total, rcount[warp] = counted;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWarps; ++i) total += rsum[i], counted += rcount[i];
        p.block_sum[blockIdx.x] = total, p.block_count[blockIdx.x] = counted;
    }
}

// ---- gradients, and the loss with them ------------------------------------------------------------
template <int BYTES>
__device__ __forceinline__ void copy_async(void *dst, const void *src, bool in) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst), n = in ? BYTES : 0;  // n = 0: fills with zeros
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}

// A tile of the whole batch, stepped by the number of blocks.  (A division per tile and warp costs
// a hundred instructions; three of them were a third of the kernel.)
struct Place {
    int n, r;  // image, tile of the image
    __device__ __forceinline__ explicit Place(const NarrowParams &p) : n((int)(blockIdx.x / p.tiles_per_image)), r((int)(blockIdx.x % p.tiles_per_image)) {}
    __device__ __forceinline__ void step(const NarrowParams &p) {
        n += p.step_images, r += p.step_tiles;
        if (r >= (int)p.tiles_per_image) r -= (int)p.tiles_per_image, ++n;
    }
    __device__ __forceinline__ bool inside(const NarrowParams &p) const { return n < (int)p.N; }
    __device__ __forceinline__ int64_t voxel() const { return (int64_t)r * kVoxels; }
};

template <typename T, bool ALIGNED, int THREADS>
__device__ __forceinline__ void fetch_tile(const NarrowParams &p, const Place &at, T *dst) {
    const int64_t v0 = at.voxel();
    const T *x = (const T *)p.x + at.n * p.sn + v0;
    const int left = (int)min((int64_t)kVoxels, p.V - v0);
    constexpr int E = ALIGNED ? 16 / (int)sizeof(T) : 1;  // aligned: V is a multiple of the vector too
    constexpr int Q = kVoxels / E, STEP = THREADS / Q;     // channels per round of the block
    const int v = threadIdx.x % Q * E;
    const bool in = v < left;
    int c = threadIdx.x / Q;
    const T *src = in ? x + c * p.sc + v : x;
    const int64_t step = in ? STEP * p.sc : 0;
    T *to = dst + c * kRow + v;
#pragma unroll 4
    for (; c < p.C; c += STEP) {
        if (ALIGNED) copy_async<16>(to, src, in);
        else if (sizeof(T) == 4) copy_async<4>(to, src, in);
        else *to = in ? *src : as_type<T>(0.f);
        src += step, to += STEP * kRow;
    }
}

__host__ __device__ inline size_t narrow_tile_bytes(int C, int esize) { return (size_t)C * kRow * esize; }
// G, weights, sums of dW, which voxels count
__host__ __device__ inline size_t narrow_fixed_bytes(int C, int OP) {
    const int rows = (C + 3) / 4 * 4, per_slot = (C + kSlots - 1) / kSlots;
    return (size_t)rows * OP * 4 + OP * 4 + 64 + (size_t)OP * kVoxels * 4 + (size_t)(per_slot * OP + 16) * kSlots * 4 + kVoxels * 4;
}

// wait until at most `n` groups of copies are under way
__device__ __forceinline__ void copies_left(int n) {
    if (n <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
}

template <typename T, int OP, bool ALIGNED, bool REG>
__global__ void __launch_bounds__(32 * kWarps, OP > 8 ? 1 : 2) narrow_kernel(const __grid_constant__ NarrowParams p) {
    constexpr int WARPS = kWarps, THREADS = 32 * WARPS;
    constexpr int GROUP = 16 / OP > 0 ? 16 / OP : 1;  // channels whose sums are reduced together
    constexpr int VW = kVoxels / WARPS;   // voxels of a warp in part 1
    constexpr int PARTS = 32 / VW;        // lanes that share a voxel
    constexpr int OL = OP / PARTS;        // labels of a lane after the reduce-scatter
    static_assert(PARTS == 4 && OP % 4 == 0, "channels and labels are dealt out to four groups of lanes");
    extern __shared__ __align__(16) float narrow_smem[];
    const int per_slot = (p.C + kSlots - 1) / kSlots, groups = REG ? 0 : (per_slot + GROUP - 1) / GROUP;
    const int rows = (p.C + 3) / 4 * 4;
    float *ws = narrow_smem;                          // [rows][OP], zeros past the last channel
    float *bs = ws + rows * OP;                       // [OP]
    float *gs = bs + OP;                              // [OP][kVoxels]
    float *sums = gs + OP * kVoxels;     // [warp][groups][32]
    int *keep = (int *)(((uintptr_t)(sums + WARPS * groups * 32) + 15) & ~(uintptr_t)15);  // [kVoxels]
    T *tiles = (T *)(keep + kVoxels);
    const int tile_elements = p.C * kRow;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    Place ahead(p);
    for (int k = 0; k + 1 < p.stages || k == 0; ++k) {
        if (ahead.inside(p)) fetch_tile<T, ALIGNED, THREADS>(p, ahead, tiles + k * tile_elements);
        ahead.step(p);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (p.stages == 1) break;
    }
    for (int i = threadIdx.x; i < rows * OP; i += THREADS) {
        const int c = i / OP, o = i % OP;
        ws[i] = o < p.O && c < p.C ? as_float<T>(((const T *)p.weight)[(int64_t)o * p.C + c]) : 0.f;
    }
    if (threadIdx.x < OP) bs[threadIdx.x] = threadIdx.x < p.O ? (p.bias ? as_float<T>(((const T *)p.bias)[threadIdx.x]) : 0.f) : -CUDART_INF_F;
    for (int i = threadIdx.x; i < WARPS * groups * 32; i += THREADS) sums[i] = 0.f;
    float factor = 1.f;
    if (p.mean && p.count_here) {
        int n = 0;
        for (int t = threadIdx.x; t < p.count_here; t += THREADS) n += p.target[t] != p.ignore;
        n = __reduce_add_sync(0xffffffffu, n);
        __shared__ int counts_s[WARPS];
        if (lane == 0) counts_s[warp] = n;
        __syncthreads();
        n = 0;
        for (int w = 0; w < WARPS; ++w) n += counts_s[w];
        factor = n ? (float)(1.0 / (double)n) : 0.f;
    } else if (p.mean) factor = p.counted ? (*p.counted ? (float)(1.0 / (double)*p.counted) : 0.f) : *p.mean_factor;
    if (p.grad_loss && !p.per_token) factor *= *p.grad_loss;
    float db[OL];
#pragma unroll
    for (int o = 0; o < OL; ++o) db[o] = 0.f;
    Pair dw[REG ? kRegisterChannels : 1][REG ? OP : 1];
    if (REG)
#pragma unroll
        for (int i = 0; i < (REG ? kRegisterChannels : 1); ++i)
#pragma unroll
            for (int o = 0; o < (REG ? OP : 1); ++o) dw[i][o] = pair(0.f, 0.f);
    double total = 0;
    int64_t count = 0;
    // this lane's voxel and labels of phase 1; the voxel's target is read a tile ahead
    const int mine = warp * VW + lane % VW, part = lane / VW;
    const auto target_of = [&](const Place &at) {
        const int64_t v = at.voxel() + mine;
        return at.inside(p) && v < p.V ? p.target[at.n * p.V + v] : p.ignore;
    };
    Place here(p);
    int64_t y_next = target_of(here);
    int stage = 0;
    while (here.inside(p)) {
        copies_left(p.stages - 2);  // this tile has landed
        __syncthreads();
        if (p.stages > 1) {
            const int into = stage == 0 ? p.stages - 1 : stage - 1;  // the tile before this one was there
            if (ahead.inside(p)) fetch_tile<T, ALIGNED, THREADS>(p, ahead, tiles + into * tile_elements);
            ahead.step(p);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const T *xs = tiles + stage * tile_elements;
        const int64_t n = here.n, v0 = here.voxel();
        here.step(p);
        {
            const int64_t y64 = y_next;
            y_next = target_of(here);
            const bool counts = v0 + mine < p.V && y64 != p.ignore;
            const int y = y64 >= 0 && y64 < p.O ? (int)y64 : -1;
            float upstream = 1.f;
            if (p.per_token && counts) upstream = p.grad_loss[n * p.V + v0 + mine];
            Pair z2[OP / 2];
#pragma unroll
            for (int o = 0; o < OP / 2; ++o) z2[o] = pair(0.f, 0.f);
            const T *row = xs + part * kRow + mine;
            const float *wrow = ws + part * OP;
            const int whole = p.C / 4, over = p.C - 4 * whole;
            const auto add = [&](const T *r, const float *wr) {
                const float v = as_float<T>(*r);
                const Pair vv = pair(v, v);
                float w[OP];
                load_weights<OP>(wr, w);
#pragma unroll
                for (int o = 0; o < OP / 2; ++o) z2[o] = fma2(pair(w[2 * o], w[2 * o + 1]), vv, z2[o]);
            };
#pragma unroll 4
            for (int i = 0; i < whole; ++i) {
                add(row, wrow);
                row += 4 * kRow, wrow += 4 * OP;
            }
            if (part < over) add(row, wrow);
            float z[OP];
#pragma unroll
            for (int o = 0; o < OP / 2; ++o) unpair(z2[o], z[2 * o], z[2 * o + 1]);
            // lane `part` ends up with the logits of labels [part * OL, (part + 1) * OL)
#pragma unroll
            for (int q = PARTS / 2; q > 0; q >>= 1) {
                const bool up = part & q;
#pragma unroll
                for (int i = 0; i < OL * q; ++i) {
                    const float mine_z = up ? z[i + OL * q] : z[i], give = up ? z[i] : z[i + OL * q];
                    z[i] = mine_z + __shfl_xor_sync(0xffffffffu, give, q * VW);
                }
            }
            float top = -CUDART_INF_F;
#pragma unroll
            for (int o = 0; o < OL; ++o) {
                z[o] += bs[part * OL + o];
                top = fmaxf(top, z[o]);
            }
#pragma unroll
            for (int q = VW; q < 32; q <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
            const float base = top == -CUDART_INF_F ? 0.f : top;
            float s = 0.f, chosen = 0.f, e[OL];
            const int hit = y - part * OL;
#pragma unroll
            for (int o = 0; o < OL; ++o) {
                e[o] = exp2_narrow((z[o] - base) * kLog2e);  // NaN logits: a NaN sum
                s += e[o];
                if (o == hit) chosen = z[o];
            }
#pragma unroll
            for (int q = VW; q < 32; q <<= 1) s += __shfl_xor_sync(0xffffffffu, s, q);
            if (counts) {
                // the lane with the target's logit adds the loss
                if ((hit >= 0 && hit < OL) || (y < 0 && part == 0)) {
                    total += y < 0 ? CUDART_NAN_F : (base - chosen) + logf(s);  // no label left: infinity - infinity
                    ++count;
                }
            }
            {
                const float g = counts ? (y < 0 ? CUDART_NAN_F : upstream * factor) : 0.f;
                const float r = g / s;
#pragma unroll
                for (int o = 0; o < OL; ++o) {
                    float d = e[o] * r;
                    if (o == hit) d -= g;
                    if (!counts || part * OL + o >= p.O) d = 0.f;
                    gs[(part * OL + o) * kVoxels + mine] = d;
                    db[o] += d;
                }
                if (part == 0) keep[mine] = counts;
            }
        }
        __syncthreads();
        {
            float g[OP][4];
            bool use[4];
            const int64_t left = p.V - v0;
#pragma unroll
            for (int o = 0; o < OP; ++o) load_voxels<float, ALIGNED>(gs + o * kVoxels, l16, g[o]);
#pragma unroll
            for (int j = 0; j < 4; ++j) use[j] = keep[voxel_of<ALIGNED>(l16, j)] != 0;
            const bool clean = __all_sync(0xffffffffu, use[0] && use[1] && use[2] && use[3]);
            T *dx = p.want_dx ? (T *)p.dx + n * p.dn + v0 + slot * p.dc : nullptr;
            const T *row = xs + slot * kRow;
            const float *wrow = ws + slot * OP;
            // one channel: dx of the lane's voxels, and the sums over them of G x added to a2
            const auto channel = [&](Pair (&a2)[OP]) {
                float v[4];
                load_voxels<T, ALIGNED>(row, l16, v);
                if (!clean) {  // what lies behind voxels that do not count reaches nothing, NaN included
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = use[j] ? v[j] : 0.f;
                }
                const Pair v01 = pair(v[0], v[1]), v23 = pair(v[2], v[3]);
                Pair d01 = pair(0.f, 0.f), d23 = d01;
                float w[OP];
                load_weights<OP>(wrow, w);
#pragma unroll
                for (int o = 0; o < OP; ++o) {
                    const Pair ww = pair(w[o], w[o]), g01 = pair(g[o][0], g[o][1]), g23 = pair(g[o][2], g[o][3]);
                    d01 = fma2(ww, g01, d01), d23 = fma2(ww, g23, d23);
                    a2[o] = fma2(v01, g01, a2[o]), a2[o] = fma2(v23, g23, a2[o]);
                }
                if (dx) {
                    float d[4];
                    unpair(d01, d[0], d[1]), unpair(d23, d[2], d[3]);
                    if (ALIGNED) {
                        Quad<T> out;
#pragma unroll
                        for (int j = 0; j < 4; ++j) out.v[j] = as_type<T>(d[j]);
                        if (4 * l16 < left) *reinterpret_cast<Quad<T> *>(dx + 4 * l16) = out;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (l16 + 16 * j < left) dx[l16 + 16 * j] = as_type<T>(d[j]);
                    }
                    dx += kSlots * p.dc;
                }
                row += kSlots * kRow, wrow += kSlots * OP;
            };
            if constexpr (REG) {
#pragma unroll
                for (int i = 0; i < kRegisterChannels; ++i)
                    if (slot + kSlots * i < p.C) channel(dw[i]);
            } else {
                for (int k = 0; k < groups; ++k) {
                    float s[16];
#pragma unroll
                    for (int q = 0; q < GROUP; ++q) {
                        Pair a2[OP];
#pragma unroll
                        for (int o = 0; o < OP; ++o) a2[o] = pair(0.f, 0.f);
                        if (slot + kSlots * (k * GROUP + q) < p.C) channel(a2);
#pragma unroll
                        for (int o = 0; o < OP; ++o) {
                            float a, b;
                            unpair(a2[o], a, b);
                            s[q * OP + o] = a + b;
                        }
                    }
                    // reduce-scatter: lane l of the half ends up with the sum over its lanes of s[l]
#pragma unroll
                    for (int w = 8; w > 0; w >>= 1) {
                        const bool up = lane & w;
#pragma unroll
                        for (int i = 0; i < w; ++i) {
                            const float mine_s = up ? s[i + w] : s[i], give = up ? s[i] : s[i + w];
                            s[i] = mine_s + __shfl_xor_sync(0xffffffffu, give, w);
                        }
                    }
                    sums[(warp * groups + k) * 32 + lane] += s[0];
                }
            }
        }
        if (p.stages == 1) {
            __syncthreads();
            if (ahead.inside(p)) fetch_tile<T, ALIGNED, THREADS>(p, ahead, tiles);
            ahead.step(p);
            asm volatile("cp.async.commit_group;" ::: "memory");
        } else if (++stage == p.stages) {
            stage = 0;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float *out = p.part + (int64_t)blockIdx.x * ((int64_t)p.O * p.C + p.O);
    __shared__ float red[WARPS][OP];
    if constexpr (REG) {
#pragma unroll
        for (int i = 0; i < kRegisterChannels; ++i)
#pragma unroll
            for (int o = 0; o < OP; ++o) {
                float a, b;
                unpair(dw[i][o], a, b);
                a += b;
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
                if (l16 == 0 && slot + kSlots * i < p.C && o < p.O) out[(int64_t)o * p.C + slot + kSlots * i] = a;
            }
    } else {
        for (int i = threadIdx.x; i < WARPS * groups * 32; i += THREADS) {
            const int w = i / (groups * 32), k = i / 32 % groups, l = i % 32;
            const int c = 2 * w + l / 16 + kSlots * (k * GROUP + l % 16 / OP), o = l % OP;
            if (c < p.C && o < p.O) out[(int64_t)o * p.C + c] = sums[i];
        }
    }
    // biases, loss and count
    __shared__ double rsum[WARPS];
    __shared__ int64_t rcount[WARPS];
#pragma unroll
    for (int o = 0; o < OL; ++o) {
        float v = db[o];
#pragma unroll
        for (int off = VW / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (lane % VW == 0) red[warp][part * OL + o] = v;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        total += __shfl_down_sync(0xffffffffu, total, off);
        count += __shfl_down_sync(0xffffffffu, count, off);
    }
    if (lane == 0) rsum[warp] = total, rcount[warp] = count;
    __syncthreads();
    if (threadIdx.x < p.O) {
        float v = 0.f;
        for (int w = 0; w < WARPS; ++w) v += red[w][threadIdx.x];
        out[(int64_t)p.O * p.C + threadIdx.x] = v;
    }
    if (threadIdx.x == 0) {
        for (int w = 1; w < WARPS; ++w) total += rsum[w], count += rcount[w];
        p.block_sum[blockIdx.x] = total, p.block_count[blockIdx.x] = count;
    }
}

}  // namespace xent
}  // namespace msd
