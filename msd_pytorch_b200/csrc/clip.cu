// Global norm over many gradient tensors, and clipping by it.
//
//   n = (sum over all tensors and elements of g^2)^(1/2)   or   max |g|
//   out = g * min(1, max_norm / (n + 1e-6))
//
// Two launches, both bound by memory: norm_kernel leaves one float64 sum per block, scale_kernel
// adds those up in every block (the same order everywhere: the same bits) and scales.  A table of the
// tensors travels in the kernel arguments; the tensors are cut into chunks of 2048 16-byte
// vectors, aligned in memory, eight vectors per thread in flight, that the blocks (four per SM, all
// resident) take in turn (a stretch of neighbouring chunks per block: 380 us instead of 311 for the
// scaling of 0.8 GB).  The second launch goes through the chunks backwards: what the first read last is
// still in L2 (everything, up to some 100 MB).
//
// An SM converts about three values per clock to float64, and HBM delivers twelve 16-bit ones.  So the
// squares of two vectors (8 or 16 values) are added pairwise in float32, and their sum is converted:
// product and three levels of sums (16-bit: exact products and four) are off by at most 4 2^-24, the
// norm by half of that.  Sums that leave float32's range are done again in float64, and float64
// tensors are float64 throughout.
//
// 0.8 GB of bfloat16: norm 136 us (5.9 TB/s), scaling into other tensors 311 us (5.1 TB/s); 96 MB of float32 in 291
// tensors: 22 and 80 us.  scale_kernel carries four types in the 64 registers that four blocks per SM leave it, and
// spills (a stack frame of 352 bytes).  Small sets are bound by the host: 88 us a call for 103 tensors.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <string.h>
#include <type_traits>
#include "common.cuh"

namespace msd {
namespace clip {

constexpr int kThreads = 256;
constexpr int kUnroll = 8;
constexpr int kChunk = kThreads * kUnroll;  // 16-byte vectors of one tensor handled by one block at a time
// Tensors per launch: the smallest table that holds them all travels (15 KB of arguments cost some
// microseconds per launch), and several launches are made for more than the largest holds.
constexpr int kTableTensors = 480, kMediumTable = 120, kSmallTable = 8;
constexpr int kBlocks = 592;                // blocks per launch, at most: four per SM

struct Entry {
    const void *in;
    void *out;
    int64_t size;
    int32_t dtype;
    int32_t first_chunk;  // of this launch
};
template <int N>
struct Table {
    int count, chunks;
    Entry e[N];
};

__host__ __device__ __forceinline__ int element_bytes(int dtype) { return dtype == MSD_F64 ? 8 : dtype == MSD_F32 ? 4 : 2; }

template <int N>
__device__ __forceinline__ int find(const Table<N> &t, int chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first_chunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double join(double a, double b, bool inf) { return inf ? (b > a || b != b ? b : a) : a + b; }

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }

// Two 16-byte vectors into the running sum.
template <typename T, bool INF>
__device__ __forceinline__ void add_vectors(const uint4 &u0, const uint4 &u1, double &acc) {
    constexpr int E = 32 / sizeof(T);
    T v[E];
    memcpy(v, &u0, 16);
    memcpy(v + E / 2, &u1, 16);
    if constexpr (sizeof(T) == 8) {
#pragma unroll
        for (int k = 0; k < E; ++k) acc = INF ? join(acc, fabs((double)v[k]), true) : fma((double)v[k], (double)v[k], acc);
    } else if constexpr (INF) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const float a = fabsf(widen<T>(v[k]));
            m = a > m || a != a ? a : m;
        }
        acc = join(acc, m, true);
    } else {
        float q[E];
#pragma unroll
        for (int k = 0; k < E; ++k) q[k] = widen<T>(v[k]) * widen<T>(v[k]);
#pragma unroll
        for (int w = E / 2; w > 0; w >>= 1)
#pragma unroll
            for (int k = 0; k < w; ++k) q[k] += q[k + w];
        if (std::is_same<T, __half>::value || (q[0] > 1e-30f && q[0] < 1e38f)) {
            acc += (double)q[0];
        } else {  // squares beyond float32's range, or nothing but zeros
            const uint32_t sign = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
            if ((u0.x | u0.y | u0.z | u0.w | u1.x | u1.y | u1.z | u1.w) & ~sign)
#pragma unroll
                for (int k = 0; k < E; ++k) acc = fma((double)widen<T>(v[k]), (double)widen<T>(v[k]), acc);
        }
    }
}

// The elements of vector `v` of a tensor whose first aligned vector holds `lead` elements of what lies
// before it: all of it, or one by one at the ends (zeros elsewhere).
template <typename T>
__device__ __forceinline__ uint4 read_vector(const T *base, int64_t v, int lead, int64_t size) {
    constexpr int E = 16 / sizeof(T);
    const int64_t i = v * E - lead;
    if (i >= 0 && i + E <= size) return *reinterpret_cast<const uint4 *>(base + i);
    T x[E];
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = i + k >= 0 && i + k < size ? base[i + k] : T(0.f);
    uint4 u;
    memcpy(&u, x, 16);
    return u;
}

template <typename T, bool INF>
__device__ __forceinline__ void norm_chunk(const Entry &e, int chunk, double &acc) {
    constexpr int E = 16 / sizeof(T);
    const int lead = (int)(((uintptr_t)e.in & 15) / sizeof(T));
    const int64_t vectors = (e.size + lead + E - 1) / E, first = (int64_t)chunk * kChunk;
    uint4 u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const int64_t v = first + k * kThreads + threadIdx.x;
        u[k] = v < vectors ? read_vector((const T *)e.in, v, lead, e.size) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; k += 2)
        if (first + k * kThreads < vectors) add_vectors<T, INF>(u[k], u[k + 1], acc);
}

__device__ __forceinline__ double block_join(double v, bool inf, double *red) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = join(v, __shfl_down_sync(0xffffffffu, v, off), inf);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kThreads / 32; ++w) v = join(v, red[w], inf);
    return v;
}

template <bool INF, int N>
__global__ void __launch_bounds__(kThreads, 4) norm_kernel(const __grid_constant__ Table<N> t, double *part) {
    __shared__ double red[kThreads / 32];
    double acc = 0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Entry &e = t.e[find(t, c)];
        const int in = c - e.first_chunk;
        switch (e.dtype) {
            case MSD_F32: norm_chunk<float, INF>(e, in, acc); break;
            case MSD_F64: norm_chunk<double, INF>(e, in, acc); break;
            case MSD_BF16: norm_chunk<__nv_bfloat16, INF>(e, in, acc); break;
            default: norm_chunk<__half, INF>(e, in, acc); break;
        }
    }
    const double s = block_join(acc, INF, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from the blocks' sums, in the same order in every block that asks.
__device__ __forceinline__ double total_norm(const double *part, int count, bool inf, double *red) {
    double n = 0;
    for (int i = threadIdx.x; i < count; i += kThreads) n = join(n, part[i], inf);
    n = block_join(n, inf, red);
    return inf ? n : sqrt(n);
}

__global__ void __launch_bounds__(kThreads) norm_finish_kernel(const double *part, int count, bool inf, float *norm32, double *norm64) {
    __shared__ double red[kThreads / 32];
    const double n = total_norm(part, count, inf, red);
    if (threadIdx.x == 0) {
        if (norm32) *norm32 = (float)n;
        if (norm64) *norm64 = n;
    }
}

// The factor, for float32 arithmetic as before * f: one factor f unless it is no normal float32 (values near
// 1e38 clipped to a small norm).  Then `before` is a power of two that leaves f near 2^-30, and what it
// makes subnormal of a value ends below the smallest float32 anyway.
struct Scale {
    double exact;
    float before, f;
    __device__ __forceinline__ explicit Scale(double v) : exact(v), before(1.f), f((float)v) {
        if (v > 0 && v < 0x1p-126) {
            const int k = min(-30 - ilogb(v), 126);
            before = scalbnf(1.f, -k), f = (float)scalbn(v, k);
        }
    }
    __device__ __forceinline__ float operator()(float v) const { return v * before * f; }
};
template <typename T>
__device__ __forceinline__ T scaled(T v, const Scale &f) {
    if constexpr (sizeof(T) == 8) return v * f.exact;
    else if constexpr (sizeof(T) == 4) return f(v);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(f(__bfloat162float(v)));
    else return __float2half_rn(f(__half2float(v)));
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const Entry &e, int chunk, const Scale &f) {
    constexpr int E = 16 / sizeof(T);
    const T *in = (const T *)e.in;
    T *out = (T *)e.out;
    const int lead = (int)(((uintptr_t)in & 15) / sizeof(T));
    const int64_t first = (int64_t)chunk * kChunk;
    if (((uintptr_t)out & 15) != ((uintptr_t)in & 15)) {  // no common alignment: one by one
        const int64_t lo = max((int64_t)0, first * E - lead), hi = min(e.size, (first + kChunk) * E - lead);
        for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) out[i] = scaled(in[i], f);
        return;
    }
    const int64_t vectors = (e.size + lead + E - 1) / E;
    uint4 u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const int64_t v = first + k * kThreads + threadIdx.x;
        if (v < vectors) u[k] = read_vector(in, v, lead, e.size);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const int64_t v = first + k * kThreads + threadIdx.x;
        if (v >= vectors) continue;
        T x[E];
        memcpy(x, &u[k], 16);
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = scaled(x[j], f);
        const int64_t i = v * E - lead;
        if (i >= 0 && i + E <= e.size) {
            memcpy(&u[k], x, 16);
            *reinterpret_cast<uint4 *>(out + i) = u[k];
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (i + j >= 0 && i + j < e.size) out[i + j] = x[j];
        }
    }
}

// Factor: min(1, max_norm / (norm + 1e-6)) of the blocks' sums, or *factor.
template <int N>
__global__ void __launch_bounds__(kThreads, 4) scale_kernel(const __grid_constant__ Table<N> t, const double *part, int parts, bool inf, double max_norm,
                                                         const float *factor, bool in_place, float *norm32, double *norm64) {
    __shared__ double red[kThreads / 32];
    double f;
    if (factor) {
        f = *factor;
        if (f == 1.0 && in_place) return;
    } else {
        const double n = total_norm(part, parts, inf, red);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            if (norm32) *norm32 = (float)n;
            if (norm64) *norm64 = n;
        }
        f = max_norm / (n + 1e-6);
        f = f > 1.0 ? 1.0 : f;
    }
    const Scale s(f);
    for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        const Entry &e = t.e[find(t, c)];
        if (f == 1.0 && e.in == e.out) continue;
        const int at = c - e.first_chunk;
        switch (e.dtype) {
            case MSD_F32: scale_chunk<float>(e, at, s); break;
            case MSD_F64: scale_chunk<double>(e, at, s); break;
            case MSD_BF16: scale_chunk<__nv_bfloat16>(e, at, s); break;
            default: scale_chunk<__half>(e, at, s); break;
        }
    }
}

// Takes tensors from `next` on into one launch's table; returns the number of chunks.
template <int N>
static int64_t fill(Table<N> *t, const msd_span_t *spans, int64_t count, int64_t *next) {
    t->count = 0;
    int64_t chunks = 0;
    while (*next < count && t->count < N) {
        const msd_span_t &s = spans[*next];
        const int E = 16 / element_bytes(s.dtype);
        const int64_t lead = (int64_t)((uintptr_t)s.data & 15) / element_bytes(s.dtype);
        const int64_t c = s.size ? ceil_div(ceil_div(s.size + lead, E), kChunk) : 0;
        if (chunks + c > 0x7fffffff) break;
        if (c) t->e[t->count++] = Entry{s.data, s.out, s.size, s.dtype, (int32_t)chunks};
        chunks += c;
        ++*next;
    }
    t->chunks = (int)chunks;
    return chunks;
}

static size_t workspace_bytes(int64_t count) { return 256 + (size_t)(ceil_div(count, kTableTensors) + 1) * kBlocks * sizeof(double); }

static int check_spans(const char *op, const msd_span_t *spans, int64_t count, bool writes) {
    if (count < 0 || (count > 0 && !spans)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: a list of tensors is needed", op);
    for (int64_t i = 0; i < count; ++i) {
        const msd_span_t &t = spans[i];
        if (t.dtype < MSD_F32 || t.dtype > MSD_F16) MSD_FAIL(MSD_ERR_UNSUPPORTED, "%s: tensor %lld has an unknown dtype %d", op, (long long)i, t.dtype);
        if (t.size < 0 || t.size >= ((int64_t)1 << 44)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: tensor %lld has a bad size", op, (long long)i);
        if (((uintptr_t)t.data | (writes ? (uintptr_t)t.out : 0)) % element_bytes(t.dtype)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: tensor %lld is not aligned to its type", op, (long long)i);
        if (t.size > 0 && (!t.data || (writes && !t.out))) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: tensor %lld has no data", op, (long long)i);
    }
    return MSD_OK;
}

template <int N>
static int launch(const msd_span_t *spans, int64_t count, bool clip, double max_norm, bool inf, float *norm32, double *norm64, double *part, cudaStream_t s) {
    Table<N> t;
    int parts = 0;
    for (int64_t next = 0; next < count;) {
        const int64_t chunks = fill(&t, spans, count, &next);
        if (!chunks) continue;
        const int blocks = (int)(chunks < kBlocks ? chunks : kBlocks);
        if (inf) norm_kernel<true, N><<<blocks, kThreads, 0, s>>>(t, part + parts);
        else norm_kernel<false, N><<<blocks, kThreads, 0, s>>>(t, part + parts);
        count_launch(true);
        MSD_CUDA_TRY(cudaGetLastError());
        parts += blocks;
    }
    if (!clip || !parts) {
        norm_finish_kernel<<<1, kThreads, 0, s>>>(part, parts, inf, norm32, norm64);
        count_launch(true);
        MSD_CUDA_TRY(cudaGetLastError());
        return MSD_OK;
    }
    const bool one_table = count <= N;  // then it is filled already
    for (int64_t next = 0; next < count;) {
        int64_t chunks = t.chunks;
        if (one_table) next = count;
        else chunks = fill(&t, spans, count, &next);
        if (!chunks) continue;
        scale_kernel<N><<<(int)(chunks < kBlocks ? chunks : kBlocks), kThreads, 0, s>>>(t, part, parts, inf, max_norm, nullptr, false, norm32, norm64);
        count_launch(true);
        MSD_CUDA_TRY(cudaGetLastError());
    }
    return MSD_OK;
}

static int run(const char *op, const msd_span_t *spans, int64_t count, bool clip, double max_norm, int norm_type, float *norm32, double *norm64, void *ws,
               size_t wsb, int device, cudaStream_t s) {
    const int rc = check_spans(op, spans, count, clip);
    if (rc) return rc;
    if (norm_type != MSD_NORM_2 && norm_type != MSD_NORM_INF) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: norm_type %d is not MSD_NORM_2 or MSD_NORM_INF", op, norm_type);
    if (clip && !(max_norm >= 0)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: max_norm must be zero or more", op);
    if (((uintptr_t)ws & 255) || !ws || wsb < workspace_bytes(count))
        MSD_FAIL(MSD_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed, %zu given", op, workspace_bytes(count), wsb);
    DeviceGuard g(device);
    MSD_CUDA_TRY(g.status);
    const bool inf = norm_type == MSD_NORM_INF;
    double *part = (double *)ws;
    if (count <= kSmallTable) return launch<kSmallTable>(spans, count, clip, max_norm, inf, norm32, norm64, part, s);
    if (count <= kMediumTable) return launch<kMediumTable>(spans, count, clip, max_norm, inf, norm32, norm64, part, s);
    return launch<kTableTensors>(spans, count, clip, max_norm, inf, norm32, norm64, part, s);
}

template <int N>
static int scale_by(const msd_span_t *spans, int64_t count, const float *factor, cudaStream_t s) {
    Table<N> t;
    bool in_place = true;
    for (int64_t i = 0; i < count; ++i) in_place = in_place && spans[i].data == spans[i].out;
    for (int64_t next = 0; next < count;) {
        const int64_t chunks = fill(&t, spans, count, &next);
        if (!chunks) continue;
        scale_kernel<N><<<(int)(chunks < kBlocks ? chunks : kBlocks), kThreads, 0, s>>>(t, nullptr, 0, false, 0.0, factor, in_place, nullptr, nullptr);
        count_launch(true);
        MSD_CUDA_TRY(cudaGetLastError());
    }
    return MSD_OK;
}

}  // namespace clip
}  // namespace msd

extern "C" MSD_API size_t msd_grad_norm_workspace_bytes(int64_t count) { return msd::clip::workspace_bytes(count < 0 ? 0 : count); }

extern "C" MSD_API int msd_grad_norm(const msd_span_t *tensors, int64_t count, int norm_type, float *norm32, double *norm64, void *workspace,
                                     size_t workspace_bytes, int device, void *stream) {
    return msd::clip::run("msd_grad_norm", tensors, count, false, 0.0, norm_type, norm32, norm64, workspace, workspace_bytes, device, (cudaStream_t)stream);
}

extern "C" MSD_API int msd_clip_grad_norm(const msd_span_t *tensors, int64_t count, double max_norm, int norm_type, float *norm32, double *norm64,
                                          void *workspace, size_t workspace_bytes, int device, void *stream) {
    return msd::clip::run("msd_clip_grad_norm", tensors, count, true, max_norm, norm_type, norm32, norm64, workspace, workspace_bytes, device,
                          (cudaStream_t)stream);
}

extern "C" MSD_API int msd_scale_tensors(const msd_span_t *tensors, int64_t count, const float *factor, int device, void *stream) {
    using namespace msd;
    using namespace msd::clip;
    if (!factor) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "msd_scale_tensors: factor must not be null");
    const int rc = check_spans("msd_scale_tensors", tensors, count, true);
    if (rc) return rc;
    DeviceGuard g(device);
    MSD_CUDA_TRY(g.status);
    if (count <= kSmallTable) return scale_by<kSmallTable>(tensors, count, factor, (cudaStream_t)stream);
    return scale_by<kTableTensors>(tensors, count, factor, (cudaStream_t)stream);
}
