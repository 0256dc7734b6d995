// Host side of the linear layer with softmax cross entropy for few labels (xent_narrow.cuh).
#include <atomic>
#include <string.h>
#include "xent_narrow.cuh"

namespace msd {

namespace fast {
int sm_count(int device);
}

namespace xent {

constexpr int kNarrowBlocks = 1184;  // of a launch, at most: 8 per SM
constexpr size_t kSmemLimit = 227 * 1024 - 1024;

// Tokens that count (an integer sum does not depend on its order).
__global__ void __launch_bounds__(1024) count_kernel(const int64_t *target, int64_t ignore, int64_t T_, unsigned long long *out) {
    __shared__ int warps[32];
    int n = 0;
    for (int64_t t = blockIdx.x * 1024ll + threadIdx.x; t < T_; t += gridDim.x * 1024ll) n += target[t] != ignore;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    n = __reduce_add_sync(0xffffffffu, warps[threadIdx.x]);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) *out = (unsigned long long)n;  // nothing has to be cleared before
        else atomicAdd(out, (unsigned long long)n);
    }
}

// Adds up the blocks' sums: 32 outputs x 8 lanes per block.  Block 0 also finishes the loss.
template <typename T>
__global__ void __launch_bounds__(256) narrow_finish_kernel(const float *part, int blocks, int64_t weights, int64_t outputs, T *dw, T *db, const double *block_sum,
                                                            const int64_t *block_count, int reduction, float *loss, float *stats) {
    __shared__ double red[8][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t i = blockIdx.x * 32ll + x;
    double s = 0;
    if (i < outputs)
        for (int b = y; b < blocks; b += 8) s += part[b * outputs + i];
    red[y][x] = s;
    __syncthreads();
    if (y == 0 && i < outputs) {
        for (int k = 1; k < 8; ++k) s += red[k][x];
        if (i < weights) {
            if (dw) dw[i] = as_type<T>((float)s);
        } else if (db) {
            db[i - weights] = as_type<T>((float)s);
        }
    }
    if (blockIdx.x == 0 && loss && y == 0) {
        double total = 0;
        int64_t count = 0;
        for (int b = x; b < blocks; b += 32) total += block_sum[b], count += block_count[b];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            total += __shfl_down_sync(0xffffffffu, total, off);
            count += __shfl_down_sync(0xffffffffu, count, off);
        }
        if (x == 0) {
            loss[0] = (float)(reduction == MSD_REDUCE_MEAN ? total / (double)count : total);
            stats[0] = reduction == MSD_REDUCE_MEAN ? (count ? (float)(1.0 / (double)count) : 0.f) : 1.f;
        }
    }
}

// Labels are padded to what the kernels are built for (the gradients' reduce-scatter needs a divisor of 32).
static int padded_labels(int64_t O, bool grad) { return O <= 4 ? 4 : O <= 8 ? 8 : O <= 12 && !grad ? 12 : 16; }

static int64_t narrow_tiles(const Problem &p) { return p.x.N * ceil_div(p.x.V, kVoxels); }

// Tiles in flight, at most four: the loads of all but one are under way while that one is worked on.
static int narrow_stages(const Problem &p) {
    const int esize = p.dtype == MSD_F32 ? 4 : 2;
    const size_t tile = narrow_tile_bytes((int)p.x.C, esize), fixed = narrow_fixed_bytes((int)p.x.C, padded_labels(p.labels, true)) + 16 + 2048;
    if (fixed >= kSmemLimit) return 0;
    // two blocks per SM where that leaves each at least two tiles
    const size_t half = kSmemLimit / 2 > fixed ? (kSmemLimit / 2 - fixed) / tile : 0;
    const size_t n = half >= 2 ? half : (kSmemLimit - fixed) / tile;
    return n > 4 ? 4 : (int)n;
}

// Where both can: two 1024 x 1024 images of 101 float32 channels, loss and gradients of 4, 8 and 16 labels 430, 600
// and 1100 us here and 3900 to 4000 as tensor-core products (tiles of 128 labels at least); one of 256 x 256, 51
// channels, 40, 44 and 51 against 138.  bfloat16, 16 labels: 1660 against 2830 us, and with 160 channels, the
// worst found, 395 against 370.
bool narrow_supported(const Problem &p) {
    return p.labels <= kNarrowLabels && p.x.sv == 1 && p.x.V >= kVoxels && p.x.C <= 1024 && p.x.N > 0 && narrow_stages(p) >= 1;
}

// 16-bit gradients are not computed ahead of the upstream gradient: they would be rounded twice,
// and a scaled float16 loss would lose those that are subnormal without its scale.
bool single_pass(const Problem &p) { return p.dtype == MSD_F32 && narrow_supported(p); }

struct NarrowSpace {
    unsigned long long *count;
    double *bsum;
    int64_t *bcount;
    float *part;
};
static size_t carve_narrow(const Problem &p, void *base, NarrowSpace *n) {
    char *b = (char *)base;
    n->count = (unsigned long long *)b;
    n->bsum = (double *)(b + 256);
    n->bcount = (int64_t *)(b + 256 + kNarrowBlocks * 8);
    n->part = (float *)(b + 256 + kNarrowBlocks * 16);
    return 256 + kNarrowBlocks * 16 + (size_t)kNarrowBlocks * (p.labels * p.x.C + p.labels) * sizeof(float);
}

size_t narrow_workspace_bytes(const Problem &p) {
    NarrowSpace n;
    return carve_narrow(p, nullptr, &n) + 256;
}

__global__ void loss_finish_kernel(const double *block_sum, const int64_t *block_count, int blocks, int reduction, float *loss, float *stats) {
    double total = 0;
    int64_t count = 0;
    for (int b = threadIdx.x; b < blocks; b += 32) total += block_sum[b], count += block_count[b];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        total += __shfl_down_sync(0xffffffffu, total, off);
        count += __shfl_down_sync(0xffffffffu, count, off);
    }
    if (threadIdx.x) return;
    if (reduction == MSD_REDUCE_MEAN) loss[0] = (float)(total / (double)count);
    if (reduction == MSD_REDUCE_SUM) loss[0] = (float)total;
    if (stats) stats[0] = reduction == MSD_REDUCE_MEAN ? (count ? (float)(1.0 / (double)count) : 0.f) : 1.f;
}

static void fill(const Problem &p, const NarrowSpace &n, NarrowParams *q) {
    memset(q, 0, sizeof(*q));
    q->x = p.x.p, q->N = p.x.N, q->V = p.x.V, q->sn = p.x.sn, q->sc = p.x.sc;
    q->C = (int)p.x.C, q->O = (int)p.labels;
    q->weight = p.weight, q->bias = p.bias, q->target = p.target, q->ignore = p.ignore_index;
    q->mean = p.reduction == MSD_REDUCE_MEAN;
    q->block_sum = n.bsum, q->block_count = n.bcount, q->part = n.part;
    q->tiles_per_image = ceil_div(p.x.V, kVoxels), q->tiles = narrow_tiles(p);
    q->stages = narrow_stages(p);
}

static bool rows_aligned(const Features &f, int esize) {
    const int64_t e = 16 / esize;
    return ((uintptr_t)f.p & 15) == 0 && f.sn % e == 0 && f.sc % e == 0 && f.V % e == 0 && f.sv == 1;
}

static int narrow_launched() {
    count_launch(true);
    MSD_CUDA_TRY(cudaGetLastError());
    return MSD_OK;
}

// Blocks of the whole GPU that can be resident together, at most one per tile.  The kernel's last answer
// (device, bytes, blocks per SM) is kept: a call of the same shape need not ask the runtime again.
template <auto KERN>
static int resident_blocks(int threads, size_t smem, int device, int64_t work, int *blocks) {
    static std::atomic<uint64_t> known, ready;
    const uint64_t last = known.load(), key = ((uint64_t)(device + 1) << 40) | (uint64_t)smem << 8;
    int per_sm = (int)(last & 255);
    if ((last & ~255ull) != key) {
        if (device >= 64 || !(ready.load() >> device & 1)) {
            MSD_CUDA_TRY(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit));
            if (device < 64) ready.fetch_or(1ull << device);
        }
        MSD_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, KERN, threads, smem));
        if (per_sm < 1) MSD_FAIL(MSD_ERR_UNSUPPORTED, "linear cross entropy: %zu bytes of shared memory do not fit", smem);
        known.store(key | (uint64_t)per_sm);
    }
    int64_t n = (int64_t)per_sm * fast::sm_count(device);
    if (n > kNarrowBlocks) n = kNarrowBlocks;
    *blocks = (int)(n < work ? n : work);
    return MSD_OK;
}

template <auto KERN>
static int launch_grad_kernel(const NarrowParams &q, size_t smem, int device, int *blocks, cudaStream_t s) {
    int rc = resident_blocks<KERN>(32 * kWarps, smem, device, q.tiles, blocks);
    if (rc) return rc;
    NarrowParams r = q;
    r.step_images = (int)(*blocks / q.tiles_per_image), r.step_tiles = (int)(*blocks % q.tiles_per_image);
    KERN<<<*blocks, 32 * kWarps, smem, s>>>(r);
    return narrow_launched();
}

template <typename T, int OP, bool ALIGNED>
static int launch_grad(const NarrowParams &q, int device, int *blocks, cudaStream_t s) {
    const size_t smem = narrow_fixed_bytes(q.C, OP) + q.stages * narrow_tile_bytes(q.C, sizeof(T)) + 16;
    if constexpr (OP <= 4)  // sums of dW in registers: 64 of them (430 us for two 1024 x 1024 images of 101 channels, 465 without)
        if (q.C <= kRegisterChannels * kSlots) return launch_grad_kernel<narrow_kernel<T, OP, ALIGNED, true>>(q, smem, device, blocks, s);
    return launch_grad_kernel<narrow_kernel<T, OP, ALIGNED, false>>(q, smem, device, blocks, s);
}

template <typename T, int OP, bool ALIGNED>
static int launch_loss(const NarrowParams &q, int device, int *blocks, cudaStream_t s) {
    const size_t smem = (size_t)q.C * OP * 8 + OP * 4;
    int rc = resident_blocks<narrow_loss_kernel<T, OP, ALIGNED>>(32 * kWarps, smem, device, ceil_div(q.N * ceil_div(q.V, 32 * loss_voxels(OP)), kWarps), blocks);
    if (rc) return rc;
    narrow_loss_kernel<T, OP, ALIGNED><<<*blocks, 32 * kWarps, smem, s>>>(q);
    return narrow_launched();
}

template <typename T, bool ALIGNED>
static int launch_narrow(const NarrowParams &q, bool grad, int device, int *blocks, cudaStream_t s) {
    switch (padded_labels(q.O, grad)) {
        case 4: return grad ? launch_grad<T, 4, ALIGNED>(q, device, blocks, s) : launch_loss<T, 4, ALIGNED>(q, device, blocks, s);
        case 8: return grad ? launch_grad<T, 8, ALIGNED>(q, device, blocks, s) : launch_loss<T, 8, ALIGNED>(q, device, blocks, s);
        case 12: return launch_loss<T, 12, ALIGNED>(q, device, blocks, s);
        default: return grad ? launch_grad<T, 16, ALIGNED>(q, device, blocks, s) : launch_loss<T, 16, ALIGNED>(q, device, blocks, s);
    }
}

static int dispatch(const Problem &p, const NarrowParams &q, bool aligned, bool grad, int device, int *blocks, cudaStream_t s) {
    if (p.dtype == MSD_F32) return aligned ? launch_narrow<float, true>(q, grad, device, blocks, s) : launch_narrow<float, false>(q, grad, device, blocks, s);
    if (p.dtype == MSD_BF16)
        return aligned ? launch_narrow<__nv_bfloat16, true>(q, grad, device, blocks, s) : launch_narrow<__nv_bfloat16, false>(q, grad, device, blocks, s);
    return aligned ? launch_narrow<__half, true>(q, grad, device, blocks, s) : launch_narrow<__half, false>(q, grad, device, blocks, s);
}

int narrow_forward(const Problem &p, float *loss, float *stats, void *ws, size_t wsb, int device, cudaStream_t s) {
    NarrowSpace n;
    const size_t need = carve_narrow(p, ws, &n);
    if (!ws || wsb < need) MSD_FAIL(MSD_ERR_WORKSPACE, "linear cross entropy forward: workspace of %zu bytes needed, %zu given", need, wsb);
    NarrowParams q;
    fill(p, n, &q);
    q.losses = p.reduction == MSD_REDUCE_NONE ? loss : nullptr;
    int blocks = 0, rc;
    if ((rc = dispatch(p, q, rows_aligned(p.x, p.dtype == MSD_F32 ? 4 : 2), false, device, &blocks, s))) return rc;
    loss_finish_kernel<<<1, 32, 0, s>>>(n.bsum, n.bcount, blocks, p.reduction, loss, stats);
    return narrow_launched();
}

int narrow_backward(const Problem &p, float *loss, float *stats, const float *grad_loss, const Features *dx, void *dw, void *db, void *ws, size_t wsb,
                    int device, cudaStream_t s) {
    NarrowSpace n;
    const size_t need = carve_narrow(p, ws, &n);
    if (!ws || wsb < need) MSD_FAIL(MSD_ERR_WORKSPACE, "linear cross entropy backward: workspace of %zu bytes needed, %zu given", need, wsb);
    const int esize = p.dtype == MSD_F32 ? 4 : 2;
    const int64_t T_ = p.x.tokens();
    NarrowParams q;
    fill(p, n, &q);
    q.grad_loss = grad_loss, q.per_token = p.reduction == MSD_REDUCE_NONE;
    q.want_dx = dx != nullptr;
    bool aligned = rows_aligned(p.x, esize);
    if (dx) {
        if (dx->sv != 1) MSD_FAIL(MSD_ERR_UNSUPPORTED, "linear cross entropy backward: the gradient's voxels must lie side by side as the features' do");
        q.dx = dx->p, q.dn = dx->sn, q.dc = dx->sc;
        aligned = aligned && rows_aligned(*dx, esize);
    }
    if (q.mean && loss && T_ <= 4096) {
        q.count_here = (int)T_;  // 16 targets a thread: less than a launch
    } else if (q.mean && loss) {
        q.counted = (const int64_t *)n.count;
        const int64_t most = (int64_t)fast::sm_count(device) * 2, blocks = T_ <= 32768 ? 1 : ceil_div(T_, 4096);
        if (blocks > 1) MSD_CUDA_TRY(cudaMemsetAsync(n.count, 0, 8, s));
        count_kernel<<<(unsigned)(blocks < most ? blocks : most), 1024, 0, s>>>(p.target, p.ignore_index, T_, n.count);
        const int rc = narrow_launched();
        if (rc) return rc;
    } else if (q.mean) {
        q.mean_factor = stats;
    }
    int blocks = 0, rc;
    if ((rc = dispatch(p, q, aligned, true, device, &blocks, s))) return rc;
    const int64_t weights = p.labels * p.x.C, outputs = weights + p.labels;
    const unsigned grid = (unsigned)ceil_div(outputs, 32);
    if (p.dtype == MSD_F32)
        narrow_finish_kernel<float><<<grid, 256, 0, s>>>(n.part, blocks, weights, outputs, (float *)dw, (float *)db, n.bsum, n.bcount, p.reduction, loss, stats);
    else if (p.dtype == MSD_BF16)
        narrow_finish_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(n.part, blocks, weights, outputs, (__nv_bfloat16 *)dw, (__nv_bfloat16 *)db, n.bsum, n.bcount,
                                                                 p.reduction, loss, stats);
    else
        narrow_finish_kernel<__half><<<grid, 256, 0, s>>>(n.part, blocks, weights, outputs, (__half *)dw, (__half *)db, n.bsum, n.bcount, p.reduction, loss,
                                                          stats);
    return narrow_launched();
}

}  // namespace xent
}  // namespace msd
