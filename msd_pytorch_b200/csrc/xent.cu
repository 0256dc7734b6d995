// Linear layer + softmax cross entropy: host side, the kernels around the products of
// xent_mma.cuh, and the C entry points.  See xent.h for the formulas.
//
// forward   pack x (and W) -> kLse -> combine (statistics, loss per token) -> finish (the reduction)
// backward  pack x (and W) -> per piece of the labels: kGrad, column sums (db), kBack (dx, dW)
#include <atomic>
#include <string.h>
#include "xent_few.cuh"
#include "xent_mma.cuh"

namespace msd {

namespace fast {
int sm_count(int device);
int make_map16(const void *ptr, int64_t cols, int64_t rows, int64_t pieces, int64_t row_stride, int64_t piece_stride, int box_rows, CUtensorMap *out);
}  // namespace fast

namespace xent {

constexpr int kThreads = 256;
constexpr int kCombineBlocks = 592;
constexpr int64_t kPieceBytes = 256ll << 20;  // G held at a time (half as much again where that saves a piece or a chunk)
constexpr int64_t kPieceLabels = 256;         // labels of a piece, at least (fewer only if there are no more)
constexpr int64_t kChunkBytes = 512ll << 20;  // packed features held at a time

static size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
static int64_t round_up(int64_t v, int64_t m) { return ceil_div(v, m) * m; }

// ---- operands ------------------------------------------------------------------------------
struct Matrix {  // row r, column c at p[(t / V) sn + (t % V) sv + c sc], t = row0 + r
    const void *p;
    int64_t rows, cols, V, sn, sv, sc;
    const int64_t *target;  // rows whose target is `ignore` count as zero; null: none
    int64_t ignore, row0;
    bool flat;  // one batch: t < V
    __device__ __forceinline__ int64_t row_start(int64_t r) const {
        const int64_t t = row0 + r;
        return flat ? t * sv : (t / V) * sn + (t % V) * sv;
    }
    __device__ __forceinline__ bool dropped(int64_t r) const { return target && target[row0 + r] == ignore; }
};

// dst[piece][row][ld] 16-bit: an operand row by row, columns past the last as zeros.  Blocks of 64
// rows x 64 columns pass through shared memory, read along whichever axis is dense.  Blocks
// [0, blocks_x) are x's, the others W's.  Three pieces: see xent_mma.cuh.
constexpr int kPackRows = 64, kPackCols = 64;
struct PackParams {
    Matrix m[2];
    uint16_t *dst[2];
    int64_t ld;
    int64_t blocks_x;
    int col_blocks;
};
// The bfloat16 next to v; the largest one where the next would be infinity.
__device__ __forceinline__ uint16_t top_piece(float v) {
    const uint16_t b = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    return (b & 0x7fff) == 0x7f80 && fabsf(v) < CUDART_INF_F ? b - 1 : b;
}
template <typename T, int P>
__global__ void __launch_bounds__(kThreads) pack_kernel(const __grid_constant__ PackParams p) {
    __shared__ T tile[kPackRows][kPackCols + 1];
    const int which = blockIdx.x < p.blocks_x ? 0 : 1;
    const int64_t block = blockIdx.x - (which ? p.blocks_x : 0);
    const Matrix &a = p.m[which];
    const int64_t r0 = block / p.col_blocks * kPackRows, c0 = block % p.col_blocks * kPackCols;
    // values first: nothing waits for targets
    if (a.sc == 1) {
        const int c = threadIdx.x % kPackCols;
        const bool in = c0 + c < a.cols;
#pragma unroll
        for (int r = threadIdx.x / kPackCols; r < kPackRows; r += kThreads / kPackCols) {
            const int64_t row = r0 + r;
            T v = T(0.f);
            if (row < a.rows && in) {
                v = ((const T *)a.p)[a.row_start(row) + c0 + c];
                if (a.dropped(row)) v = T(0.f);
            }
            tile[r][c] = v;
        }
    } else {
        const int r = threadIdx.x % kPackRows;
        const int64_t row = r0 + r;
        const bool in = row < a.rows;
        const T *src = (const T *)a.p + (in ? a.row_start(row) : 0) + c0 * a.sc;
        T v[kPackCols / (kThreads / kPackRows)];
#pragma unroll
        for (int k = 0; k < kPackCols / (kThreads / kPackRows); ++k) {
            const int c = threadIdx.x / kPackRows + k * (kThreads / kPackRows);
            v[k] = in && c0 + c < a.cols ? src[c * a.sc] : T(0.f);
        }
        const bool drop = in && a.dropped(row);
#pragma unroll
        for (int k = 0; k < kPackCols / (kThreads / kPackRows); ++k) tile[r][threadIdx.x / kPackRows + k * (kThreads / kPackRows)] = drop ? T(0.f) : v[k];
    }
    __syncthreads();
    const int64_t piece = a.rows * p.ld;
    const int c = threadIdx.x % (kPackCols / 4) * 4;  // ld is a multiple of 8: four columns are all in or all out
    const int64_t col = c0 + c;
    if (col >= p.ld) return;
#pragma unroll
    for (int r = threadIdx.x / (kPackCols / 4); r < kPackRows; r += kThreads / (kPackCols / 4)) {
        const int64_t row = r0 + r;
        if (row >= a.rows) break;
        uint16_t *out = p.dst[which] + row * p.ld + col;
        if constexpr (P == 3) {
            uint16_t h[3][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = (float)tile[r][c + k];
                h[0][k] = top_piece(v);
                const float d = fabsf(v) < CUDART_INF_F ? v - __bfloat162float(__ushort_as_bfloat16(h[0][k])) : 0.f;  // infinities have one piece
                const __nv_bfloat16 m = __float2bfloat16_rn(d);
                h[1][k] = __bfloat16_as_ushort(m), h[2][k] = __bfloat16_as_ushort(__float2bfloat16_rn(d - __bfloat162float(m)));
            }
#pragma unroll
            for (int i = 0; i < 3; ++i)
                *reinterpret_cast<uint2 *>(out + i * piece) = make_uint2((uint32_t)h[i][0] | ((uint32_t)h[i][1] << 16), (uint32_t)h[i][2] | ((uint32_t)h[i][3] << 16));
        } else {
            uint16_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) memcpy(h + k, &tile[r][c + k], 2);
            *reinterpret_cast<uint2 *>(out) = make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
        }
    }
}

// The reduced loss, and behind the log-sum-exps the factor of the reduction.
__device__ __forceinline__ void finish_loss(double total, int64_t count, int reduction, float *loss, const Stats &stats) {
    if (reduction == MSD_REDUCE_MEAN) loss[0] = (float)(total / (double)count);
    if (reduction == MSD_REDUCE_SUM) loss[0] = (float)total;
    if (stats.lse) *stats.factor = reduction == MSD_REDUCE_MEAN ? (count ? (float)(1.0 / (double)count) : 0.f) : 1.f;
}

// ---- forward: joining the tiles, reducing the losses ---------------------------------------------
// Joins the (maximum, sum) pairs of all label tiles: statistics and loss of every token;
// per block the sum of the losses and the number of tokens that count.  TX tokens x 256 / TX lanes.  A
// block that is the only one finishes the loss too.
template <int TX>
__global__ void __launch_bounds__(kThreads) combine_kernel(const float2 *part, const float *zy, const int64_t *target, int64_t ignore, int64_t T_, int64_t O,
                                                           int slots, const Stats stats, float *losses, double *block_sum, int64_t *block_count, int reduction,
                                                           float *loss) {
    constexpr int LANES = kThreads / TX;
    __shared__ float2 red[LANES][TX + 1];
    __shared__ double ssum[TX];
    __shared__ int64_t scount[TX];
    double total = 0;
    int64_t count = 0;
    const int x = threadIdx.x % TX, w = threadIdx.x / TX;
    const auto join = [](float &m, float &s, const float2 &v) {
        const float up = fmaxf(m, v.x), base = up == -CUDART_INF_F ? 0.f : up;
        s = s * exp2f((m - base) * kLog2e) + v.y * exp2f((v.x - base) * kLog2e);
        m = up;
    };
    for (int64_t t0 = blockIdx.x * (int64_t)TX; t0 < T_; t0 += gridDim.x * (int64_t)TX) {
        const int64_t t = t0 + x;
        float m = -CUDART_INF_F, s = 0.f;
        if (t < T_) {
#pragma unroll 4
            for (int i = w; i < slots; i += LANES) join(m, s, part[i * T_ + t]);
        }
        red[w][x] = make_float2(m, s);
        __syncthreads();
#pragma unroll
        for (int h = LANES / 2; h >= 8; h >>= 1) {  // the last eight in order
            if (w < h) {
                join(m, s, red[w + h][x]);
                red[w][x] = make_float2(m, s);
            }
            __syncthreads();
        }
        if (w == 0 && t < T_) {
            for (int i = 1; i < 8; ++i) join(m, s, red[i][x]);
            const float log_s = logf(s);
            const int64_t y = target[t];
            float loss = 0.f;
            if (y != ignore) {
                loss = y >= 0 && y < O ? (m - zy[t]) + log_s : CUDART_NAN_F;  // NaN: a target that names no label
                ++count;
            }
            if (stats.lse) stats.write(t, m, log_s);
            if (losses) losses[t] = loss;
            total += loss;
        }
        __syncthreads();
    }
    if (w == 0) ssum[x] = total, scount[x] = count;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < TX; ++i) total += ssum[i], count += scount[i];
        if (gridDim.x == 1 && loss) finish_loss(total, count, reduction, loss, stats);
        else block_sum[blockIdx.x] = total, block_count[blockIdx.x] = count;
    }
}

__global__ void __launch_bounds__(kThreads) finish_kernel(const double *block_sum, const int64_t *block_count, int blocks, int reduction, float *loss,
                                                          const Stats stats) {
    __shared__ double ssum[kThreads];
    __shared__ int64_t scount[kThreads];
    double total = 0;
    int64_t count = 0;
    for (int i = threadIdx.x; i < blocks; i += kThreads) total += block_sum[i], count += block_count[i];
    ssum[threadIdx.x] = total, scount[threadIdx.x] = count;
    __syncthreads();
    for (int w = kThreads / 2; w > 0; w >>= 1) {
        if (threadIdx.x < w) ssum[threadIdx.x] += ssum[threadIdx.x + w], scount[threadIdx.x] += scount[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x) return;
    total = ssum[0], count = scount[0];
    finish_loss(total, count, reduction, loss, stats);
}

// ---- backward ------------------------------------------------------------------------------
__device__ __forceinline__ void store(void *p, int type, int64_t i, float v) {
    if (type == MSD_F32) ((float *)p)[i] = v;
    else if (type == MSD_BF16) ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
    else ((__half *)p)[i] = __float2half_rn(v);
}

// db: the sums over 32 tokens each that kGrad left, added in float64.  X labels x 1024 / X lanes.
// `run`: sums of earlier chunks of the tokens (add) and for later ones (not last).
template <int X>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float *columns, int64_t width, int64_t labels, int64_t rows, const Factor factor, float g_scale,
                                                          int type, void *db, double *run, bool add, bool last) {
    constexpr int LANES = 1024 / X;
    __shared__ double red[LANES][X + 1];
    const int x = threadIdx.x % X, y = threadIdx.x / X;
    const int64_t o = blockIdx.x * (int64_t)X + x;
    double s = 0;
    if (o < labels) {
#pragma unroll 4
        for (int64_t i = y; i < rows; i += LANES) s += columns[i * width + o];
    }
    red[y][x] = s;
    __syncthreads();
#pragma unroll
    for (int h = LANES / 2; h >= 16; h >>= 1) {
        if (y < h) red[y][x] += red[y + h][x];
        __syncthreads();
    }
    if (y == 0 && o < labels) {
        s = red[0][x];
        for (int i = 1; i < 16; ++i) s += red[i][x];
        if (add) s += run[o];
        if (last) store(db, type, o, (float)s / g_scale * factor.value());
        else run[o] = s;
    }
}

// Joins the ranges of a split contraction in order: 32 results x 8 lanes per block, or, with few
// ranges, a thread per result.
constexpr int kFewSplits = 8;
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ MmaParams p, int which, int out_type) {
    __shared__ double red[8][33];
    const Product &q = p.p[which];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const bool few = q.splits <= kFewSplits;
    const int64_t i = few ? blockIdx.x * (int64_t)kThreads + threadIdx.x : blockIdx.x * 32ll + x;
    const bool in = i < (int64_t)q.M * q.N;
    // along whichever axis of the result is dense
    const bool by_column = q.sc == 1;
    const int64_t m = by_column ? i / q.N : i % q.M, n = by_column ? i % q.N : i / q.M, j = m * q.ld + n;
    double s = 0;
    if (in) {
#pragma unroll 4
        for (int k = few ? 0 : y; k < q.splits; k += few ? 1 : 8) s += q.part[(int64_t)k * q.M * q.ld + j];
    }
    if (!few) {
        red[y][x] = s;
        __syncthreads();
        if (y) return;
        for (int k = 1; k < 8; ++k) s += red[k][x];
    }
    if (!in) return;
    if (q.add) s += q.sum[j];
    if (!q.last) {
        q.sum[j] = (float)s;
        return;
    }
    store(q.out, out_type, ((q.row0 + m) / q.V) * q.sn + ((q.row0 + m) % q.V) * q.sm + n * q.sc, (float)s * (p.factor.value() / p.g_scale));
}

// ---- host -----------------------------------------------------------------------------------
struct Plan {
    int P;               // pieces of an operand
    bool joins;          // 16-bit gradients of products in pieces: always in partial sums that are joined
    int64_t T, C, O, ld;  // tokens, channels, labels, channels as packed
    bool pack_w;
    int64_t chunk, chunks;  // tokens at a time: neither more than 512 MB of packed features, nor a piece of G above its limit
    int64_t pieces, width;  // label pieces of the backward pass
};

// `backward`: of the products with G.  Weights per token may span many orders of magnitude, and one float16
// holds G over few of them: with such weights float16 goes through the three pieces too.
static Plan make_plan(const Problem &p, bool backward) {
    Plan q;
    q.P = p.dtype == MSD_F32 || (backward && p.dtype == MSD_F16 && p.reduction == MSD_REDUCE_NONE) ? 3 : 1;
    q.joins = q.P > 1 && p.dtype != MSD_F32;
    q.T = p.x.tokens(), q.C = p.x.C, q.O = p.labels;
    q.ld = round_up(q.C, 8);
    q.pack_w = q.P > 1 || q.C % 8 || ((uintptr_t)p.weight & 15);
    const int64_t g_labels = q.O < kPieceLabels ? round_up(q.O, 64) : kPieceLabels;
    const int64_t by_x = kChunkBytes / (2 * q.P * q.ld), by_g = kPieceBytes / (2 * q.P * g_labels);
    q.chunk = (by_x < by_g ? by_x : by_g) / kTileM * kTileM;
    if (q.T <= by_g + by_g / 2 && q.T <= by_x) q.chunk = q.T;
    if (q.chunk < 16 * kTileM) q.chunk = 16 * kTileM;
    if (q.chunk > q.T) q.chunk = q.T;
    q.chunks = q.T ? ceil_div(q.T, q.chunk) : 0;
    const int64_t per_label = (q.T ? q.chunk : 1) * 2 * q.P;
    int64_t most = kPieceBytes / per_label;
    if (most < kPieceLabels) most = kPieceLabels;
    q.pieces = (q.O + most / 2) / most;
    if (q.pieces < 1) q.pieces = 1;
    q.width = round_up(ceil_div(q.O, q.pieces), 64);
    q.pieces = ceil_div(q.O, q.width);
    return q;
}

// Hands out pieces of the workspace; with a null base it only counts.
struct Carver {
    char *base;
    size_t used = 0;
    explicit Carver(void *p) : base((char *)p) {}
    template <typename T>
    T *take(size_t count) {
        T *r = (T *)(base ? base + used : nullptr);
        used += pad256(count * sizeof(T));
        return r;
    }
};

struct Operands {
    uint16_t *x, *w;
};

static Operands carve_operands(const Plan &q, Carver *c) {
    Operands o;
    o.x = c->take<uint16_t>(q.P * q.chunk * q.ld);
    o.w = q.pack_w ? c->take<uint16_t>(q.P * q.O * q.ld) : nullptr;
    return o;
}

// What the forward call leaves to the backward call: log-sum-exps and the reduction's factor, and,
// unless they are large, the packed operands.
constexpr size_t kKeptBytes = 256u << 20;
static size_t stats_bytes(const Plan &q) { return Stats::bytes(q.T); }
static bool keeps_operands(const Plan &q) {
    Carver c(nullptr);
    carve_operands(q, &c);
    return q.chunks <= 1 && c.used <= kKeptBytes;
}

struct ForwardSpace {
    float2 *part;
    float *zy;
    double *bsum;
    int64_t *bcount;
};
static ForwardSpace carve_forward(const Plan &q, Carver *c) {
    ForwardSpace f;
    const int64_t slots = 2 * ceil_div(q.O, 128);  // two per tile, tiles of 128 labels and more
    f.part = c->take<float2>((q.T <= kFewTokens && slots < kFewBlocks ? kFewBlocks : slots) * q.chunk);
    f.zy = c->take<float>(q.chunk);
    f.bsum = c->take<double>(kCombineBlocks * q.chunks);
    f.bcount = c->take<int64_t>(kCombineBlocks * q.chunks);
    return f;
}

struct BackwardSpace {
    uint16_t *g;
    float *run, *columns, *part[2];
    float *run_w;    // several chunks: sums of dW and db
    double *run_b;
};

// Contraction ranges of the two products of one backward launch: a product is split when one
// of its tiles alone would outlast the average load of a pair of SMs.
static void choose_splits(const Plan &q, int64_t tokens, int64_t labels, int pairs, int *sx, int *sw) {
    const int64_t kx = ceil_div(labels, kDepth), kw = ceil_div(tokens, kDepth);
    const int64_t tn = ceil_div(q.C, kTileN), tx = ceil_div(tokens, kTileM) * tn, tw = ceil_div(labels, kTileM) * tn;
    int64_t share = ceil_div(tx * kx + tw * kw, pairs);
    if (share < 4) share = 4;
    *sx = (int)ceil_div(kx, share), *sw = (int)ceil_div(kw, share);
}

static BackwardSpace carve_backward(const Plan &q, Carver *c) {
    BackwardSpace b;
    b.g = c->take<uint16_t>(q.P * q.chunk * q.width);
    const int64_t ld = round_up(q.C, 4);
    b.run = q.pieces > 1 ? c->take<float>(q.chunk * ld) : nullptr;
    b.run_w = q.chunks > 1 ? c->take<float>(q.O * ld) : nullptr;
    b.run_b = q.chunks > 1 ? c->take<double>(q.O) : nullptr;
    b.columns = c->take<float>(ceil_div(q.chunk, 32) * q.width);
    size_t most[2] = {0, 0};
    // chunks and pieces in the middle are like the first
    const int64_t tokens[2] = {q.chunk, q.T - (q.chunks - 1) * q.chunk}, labels[2] = {q.O < q.width ? q.O : q.width, q.O - (q.pieces - 1) * q.width};
    for (int i = 0; i < 4; ++i) {
        const int64_t t = tokens[i & 1], w = labels[i >> 1];
        int s[2];
        choose_splits(q, t, w, kMaxPairs, &s[0], &s[1]);
        const size_t n[2] = {s[0] > 1 || q.joins ? (size_t)s[0] * t * ld : 0, s[1] > 1 || q.joins ? (size_t)s[1] * w * ld : 0};
        for (int k = 0; k < 2; ++k) most[k] = n[k] > most[k] ? n[k] : most[k];
    }
    for (int i = 0; i < 2; ++i) b.part[i] = most[i] ? c->take<float>(most[i]) : nullptr;
    return b;
}

size_t forward_workspace_bytes(const Problem &p) {
    if (narrow_supported(p)) return narrow_workspace_bytes(p);
    Carver c(nullptr);
    const Plan q = make_plan(p, false);
    carve_forward(q, &c);
    carve_operands(q, &c);
    return c.used + 256;
}

// Whether the forward call left the operands as the backward call takes them.  (few_forward packs none.)
static bool kept_by_forward(const Problem &p, const Plan &backward) {
    const Plan f = make_plan(p, false);
    return f.P == backward.P && keeps_operands(f) && !few_supported(p);
}

// Enough for every reduction.
size_t backward_workspace_bytes(const Problem &p) {
    if (narrow_supported(p)) return narrow_workspace_bytes(p);
    size_t most = 0;
    Problem r = p;
    for (int reduction : {MSD_REDUCE_NONE, MSD_REDUCE_MEAN}) {
        r.reduction = reduction;
        Carver c(nullptr);
        const Plan q = make_plan(r, true);
        carve_backward(q, &c);
        if (!kept_by_forward(r, q)) carve_operands(q, &c);
        if (c.used > most) most = c.used;
    }
    return most + 256;
}

size_t saved_bytes(const Problem &p) {
    const Plan q = make_plan(p, false);
    if (narrow_supported(p)) return 256;
    if (few_supported(p)) return stats_bytes(q);
    Carver c(nullptr);
    if (keeps_operands(q)) carve_operands(q, &c);
    return stats_bytes(q) + c.used;
}

static int pair_count(int sms) { return sms / 2 < 1 ? 1 : sms / 2 > kMaxPairs ? kMaxPairs : sms / 2; }

static int launched() {
    count_launch(true);
    MSD_CUDA_TRY(cudaGetLastError());
    return MSD_OK;
}
#define XENT_TRY(expr)           \
    do {                         \
        const int rc__ = (expr); \
        if (rc__) return rc__;   \
    } while (0)

// Packs the tokens [t0, t0 + n) of x and, with the first of them, W where needed.
static int pack_operands(const Problem &p, const Plan &q, const Operands &op, int64_t t0, int64_t n, cudaStream_t s) {
    PackParams k;
    k.m[0] = Matrix{p.x.p, n, q.C, p.x.V, p.x.sn, p.x.sv, p.x.sc, p.target, p.ignore_index, t0, p.x.N == 1};
    k.m[1] = Matrix{p.weight, q.O, q.C, q.O, 0, q.C, 1, nullptr, 0, 0, true};
    k.dst[0] = op.x, k.dst[1] = op.w;
    k.ld = q.ld;
    k.col_blocks = (int)ceil_div(q.ld, kPackCols);
    const int64_t bx = ceil_div(n, kPackRows) * k.col_blocks, bw = q.pack_w && t0 == 0 ? ceil_div(q.O, kPackRows) * k.col_blocks : 0;
    if (bx + bw > 0x7fffffff) MSD_FAIL(MSD_ERR_UNSUPPORTED, "linear cross entropy: %lld labels times %lld channels are too many", (long long)q.O, (long long)q.C);
    k.blocks_x = bx;
    const unsigned grid = (unsigned)(bx + bw);
    if (p.dtype == MSD_F32) pack_kernel<float, 3><<<grid, kThreads, 0, s>>>(k);
    else if (q.P > 1) pack_kernel<__half, 3><<<grid, kThreads, 0, s>>>(k);
    else if (p.dtype == MSD_BF16) pack_kernel<__nv_bfloat16, 1><<<grid, kThreads, 0, s>>>(k);
    else pack_kernel<__half, 1><<<grid, kThreads, 0, s>>>(k);
    return launched();
}

template <int USE>
static int launch_mma(const MmaParams &m, int P, bool run, int pairs, cudaStream_t s) {
    const int which = P > 1 ? 2 : run;
    auto kern = which == 2 ? xent_mma_kernel<USE, 3, true> : which ? xent_mma_kernel<USE, 1, true> : xent_mma_kernel<USE, 1, false>;
    const size_t smem = mma_smem_bytes(P);
    static std::atomic<uint64_t> ready[3];  // devices whose kernel is set up
    int device = 0;
    MSD_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 64 || !(ready[which].load() >> device & 1)) {
        if (which) {
            cudaFuncAttributes a;
            MSD_CUDA_TRY(cudaFuncGetAttributes(&a, kern));
            if (a.numRegs < kRegsLaunch) MSD_FAIL(MSD_ERR_UNSUPPORTED, "linear cross entropy: built with %d registers per thread, %d expected", a.numRegs, kRegsLaunch);
        }
        MSD_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (device < 64) ready[which].fetch_or(1ull << device);
    }
    kern<<<2 * pairs, kMmaThreads, smem, s>>>(m);
    return launched();
}

// What the three uses have in common.
static int common_params(const Problem &p, const Plan &q, const Operands &op, int64_t t0, int device, MmaParams *m) {
    memset(m, 0, sizeof(*m));
    m->bf16 = p.dtype == MSD_BF16 || q.P > 1;
    m->bias = p.bias, m->bias_type = p.dtype;
    m->target = p.target + t0, m->ignore = p.ignore_index, m->labels = (int)q.O;
    m->group_m = 64;  // 8192 rows of x: 16 MB at 1024 channels
    m->status = tma::device_status_ptr(device);
    if (!m->status) MSD_FAIL(MSD_ERR_CUDA, "linear cross entropy: cannot locate the status word");
    return MSD_OK;
}

// z = x W^T of `tokens` packed tokens over the labels [label0, label0 + n)
static int logit_product(const Problem &p, const Plan &q, const Operands &op, int64_t tokens, int64_t label0, int64_t n, int pairs, Product *r) {
    r->M = (int)tokens, r->N = (int)n, r->K = (int)q.C;
    r->tiles_m = (int)ceil_div(tokens, kTileM);
    // the width whose rounds over all pairs take the least time (1023 x 10007: three rounds of 192
    // instead of three of 256)
    int64_t best = 0;
    for (int w = kTileN; w >= 128; w -= 64) {
        const int64_t cost = ceil_div(r->tiles_m * ceil_div(n, w), pairs) * (w + 16);
        if (w == kTileN || cost < best) best = cost, r->tile_n = w;
    }
    r->tiles_n = (int)ceil_div(n, r->tile_n);
    r->splits = 1, r->k_blocks = (int)ceil_div(q.C, kDepth);
    const uint16_t *w = q.pack_w ? op.w : (const uint16_t *)p.weight;
    if ((int64_t)r->tiles_m * r->tiles_n > 0x7fffffff) MSD_FAIL(MSD_ERR_UNSUPPORTED, "linear cross entropy: %lld tokens times %lld labels are too many", (long long)tokens, (long long)n);
    XENT_TRY(fast::make_map16(op.x, q.ld, tokens, q.P, q.ld, tokens * q.ld, kCtaM, &r->a));
    return fast::make_map16(w + label0 * q.ld, q.ld, n, q.P, q.ld, q.O * q.ld, kCtaN, &r->b);
}

// Few tokens: every label's row of W is read once, straight from memory.
static int few_forward(const Problem &p, float *loss, float *saved, float2 *part, float *zy, int device, cudaStream_t s) {
    FewParams f;
    f.x = p.x, f.weight = p.weight, f.bias = p.bias, f.target = p.target, f.ignore = p.ignore_index;
    f.T = (int)p.x.tokens(), f.O = p.labels, f.part = part, f.zy = zy;
    const int esize = p.dtype == MSD_F32 ? 4 : 2;
    f.vec = p.x.C % (16 / esize) == 0 && ((uintptr_t)p.weight & 15) == 0;
    f.C4 = (int)round_up(p.x.C, 256);
    const int64_t groups = ceil_div(p.labels, kFewRows * kFewWarps), all = 2 * (int64_t)fast::sm_count(device), most = all < kFewBlocks ? all : kFewBlocks;
    const int blocks = (int)(groups < most ? groups : most);
    int rc;
    if (p.dtype == MSD_F32) rc = launch_few<float>(f, blocks, s);
    else if (p.dtype == MSD_BF16) rc = launch_few<__nv_bfloat16>(f, blocks, s);
    else rc = launch_few<__half>(f, blocks, s);
    if (rc) return rc;
    count_launch(true);
    few_finish_kernel<<<1, 32 * kFewTokens, 0, s>>>(part, zy, p.target, p.ignore_index, f.T, p.labels, blocks, p.reduction, loss, Stats::of(saved, f.T));
    return launched();
}

int forward(const Problem &p, float *loss, float *saved, void *ws, size_t wsb, int device, cudaStream_t s) {
    if (narrow_supported(p)) return narrow_forward(p, loss, saved, ws, wsb, device, s);
    const Plan q = make_plan(p, false);
    Carver c(ws);
    const ForwardSpace f = carve_forward(q, &c);
    Operands op = carve_operands(q, &c);
    if (!ws || wsb < c.used) MSD_FAIL(MSD_ERR_WORKSPACE, "linear cross entropy forward: workspace of %zu bytes needed, %zu given", c.used, wsb);
    if (few_supported(p) && q.T) return few_forward(p, loss, saved, f.part, f.zy, device, s);
    if (saved && keeps_operands(q)) {
        Carver k((char *)saved + stats_bytes(q));
        op = carve_operands(q, &k);
    }
    const int sms = fast::sm_count(device), pairs = pair_count(sms);
    const Stats stats = Stats::of(saved, q.T);
    int64_t blocks = 0;
    bool alone = false;
    for (int64_t t0 = 0; t0 < q.T; t0 += q.chunk) {
        const int64_t n = q.T - t0 < q.chunk ? q.T - t0 : q.chunk;
        XENT_TRY(pack_operands(p, q, op, t0, n, s));
        MmaParams m;
        XENT_TRY(common_params(p, q, op, t0, device, &m));
        XENT_TRY(logit_product(p, q, op, n, 0, q.O, pairs, &m.p[0]));
        m.part = f.part, m.zy = f.zy;
        const int64_t tiles = (int64_t)m.p[0].tiles_m * m.p[0].tiles_n;
        m.sum_blocks = !saved && tiles <= pairs ? kSumSmall : kSumStep;
        XENT_TRY(launch_mma<kLse>(m, q.P, m.p[0].k_blocks > m.sum_blocks, (int)(tiles < pairs ? tiles : pairs), s));
        // many lanes per token where there are few tokens: their pairs would be joined one after the other
        const int slots = 2 * m.p[0].tiles_n;
        alone = q.chunks == 1 && n * slots <= 8192;  // one block's work is less than a launch
        const int tx = !alone && n <= 4096 ? 4 : 32;
        const int64_t more = alone ? 1 : ceil_div(n, tx) < kCombineBlocks ? ceil_div(n, tx) : kCombineBlocks;
        auto combine = tx == 4 ? combine_kernel<4> : combine_kernel<32>;
        combine<<<(unsigned)more, kThreads, 0, s>>>(f.part, f.zy, p.target + t0, p.ignore_index, n, q.O, slots, stats.at(t0),
                                                   p.reduction == MSD_REDUCE_NONE ? loss + t0 : nullptr, f.bsum + blocks, f.bcount + blocks, p.reduction, alone ? loss : nullptr);
        XENT_TRY(launched());
        blocks += more;
    }
    if (alone) return MSD_OK;
    finish_kernel<<<1, kThreads, 0, s>>>(f.bsum, f.bcount, (int)blocks, p.reduction, loss, stats);
    return launched();
}

// Contiguous ranges of items for every pair: the items of product 0 evenly, then those of product 1
// so that the loads level out.
static void assign(MmaParams *m, int pairs, bool use0, bool use1) {
    const int64_t n0 = use0 ? (int64_t)m->p[0].tiles_m * m->p[0].tiles_n * m->p[0].splits : 0;
    const int64_t n1 = use1 ? (int64_t)m->p[1].tiles_m * m->p[1].tiles_n * m->p[1].splits : 0;
    const double c0 = use0 ? (double)m->p[0].k_blocks / m->p[0].splits + 1 : 0, c1 = use1 ? (double)m->p[1].k_blocks / m->p[1].splits + 1 : 1;
    int64_t load0[kMaxPairs];
    m->first[0][0] = m->first[1][0] = 0;
    for (int i = 0; i < pairs; ++i) {
        load0[i] = n0 * (i + 1) / pairs - n0 * i / pairs;
        m->first[0][i + 1] = (int)(n0 * (i + 1) / pairs);
    }
    const auto room = [&](double level, int i) {
        const double r = (level - load0[i] * c0) / c1;
        return r > 0 ? (int64_t)r : (int64_t)0;
    };
    double lo = 0, hi = n0 * c0 + n1 * c1 + c1;
    for (int it = 0; it < 60; ++it) {  // the smallest level that holds everything
        const double mid = 0.5 * (lo + hi);
        int64_t held = 0;
        for (int i = 0; i < pairs; ++i) held += room(mid, i);
        if (held >= n1) hi = mid;
        else lo = mid;
    }
    int64_t at = 0;
    for (int i = 0; i < pairs; ++i) {
        at += room(hi, i);
        if (at > n1) at = n1;
        m->first[1][i + 1] = (int)at;
    }
    m->first[1][pairs] = (int)n1;
}

// Gradients from the tokens [t0, t0 + T_) and the labels [o0, o0 + width): G, then the sums over it.
static int backward_piece(const Problem &p, const Plan &q, const Operands &op, const BackwardSpace &b, const Stats &stats, const float *row_factor, const Factor &factor,
                          int64_t t0, int64_t T_, int64_t o0, const Features *dx, void *dw, void *db, int device, int pairs, cudaStream_t s) {
    const size_t esize = p.dtype == MSD_F32 ? 4 : 2;
    const int64_t n = q.O - o0 < q.width ? q.O - o0 : q.width, gw = round_up(n, 64), g_piece = T_ * gw;
    const uint16_t *w = q.pack_w ? op.w : (const uint16_t *)p.weight;
    const bool first = t0 == 0, last = t0 + T_ == q.T;
    MmaParams m;
    XENT_TRY(common_params(p, q, op, t0, device, &m));
    XENT_TRY(logit_product(p, q, op, T_, o0, n, pairs, &m.p[0]));
    m.label0 = (int)o0, m.sum_blocks = kSumStep;
    m.stats = stats.at(t0), m.row_factor = row_factor ? row_factor + t0 : nullptr, m.factor = factor;
    m.columns = db ? b.columns : nullptr;
    m.g = b.g, m.g_width = gw, m.g_piece = g_piece;
    // |G| <= 2 in units of the factor: one float16 holds it times 2^14, down to 2^-38
    m.g_scale = p.dtype == MSD_F16 && q.P == 1 ? 16384.f : 1.f;
    const int64_t tiles = (int64_t)m.p[0].tiles_m * m.p[0].tiles_n;
    XENT_TRY(launch_mma<kGrad>(m, q.P, m.p[0].k_blocks > m.sum_blocks, (int)(tiles < pairs ? tiles : pairs), s));
    if (db) {
        const int x = n < 1024 ? 8 : 32;  // few labels: more lanes for each
        auto sum = x == 8 ? column_sum_kernel<8> : column_sum_kernel<32>;
        sum<<<(unsigned)ceil_div(n, x), 1024, 0, s>>>(b.columns, gw, n, ceil_div(T_, 32), factor, m.g_scale, p.dtype, (char *)db + o0 * esize,
                                                      b.run_b ? b.run_b + o0 : nullptr, !first, last);
        XENT_TRY(launched());
    }
    if (!dx && !dw) return MSD_OK;
    int splits[2];
    choose_splits(q, T_, n, kMaxPairs, &splits[0], &splits[1]);
    Product &X = m.p[0], &W = m.p[1];
    X.M = (int)T_, X.N = (int)q.C, X.K = (int)n;
    X.a_mn = false, X.b_mn = true;
    X.sum = b.run, X.add = o0 > 0, X.last = o0 + n >= q.O;
    X.V = q.T, X.sc = 1, X.row0 = t0;
    if (dx) X.out = dx->p, X.V = dx->V, X.sn = dx->sn, X.sm = dx->sv, X.sc = dx->sc;
    XENT_TRY(fast::make_map16(b.g, gw, T_, q.P, gw, g_piece, kCtaM, &X.a));
    XENT_TRY(fast::make_map16(w + o0 * q.ld, q.ld, n, q.P, q.ld, q.O * q.ld, kDepth, &X.b));
    W.M = (int)n, W.N = (int)q.C, W.K = (int)T_;
    W.a_mn = true, W.b_mn = true;
    W.sum = b.run_w ? b.run_w + o0 * round_up(q.C, 4) : nullptr, W.add = !first, W.last = last;
    W.out = (char *)dw + o0 * q.C * esize, W.V = n, W.sm = q.C, W.sc = 1;
    XENT_TRY(fast::make_map16(b.g, gw, T_, q.P, gw, g_piece, kDepth, &W.a));
    XENT_TRY(fast::make_map16(op.x, q.ld, T_, q.P, q.ld, T_ * q.ld, kDepth, &W.b));
    for (int i = 0; i < 2; ++i) {
        Product &r = m.p[i];
        r.tile_n = kTileN;
        r.tiles_m = (int)ceil_div(r.M, kTileM), r.tiles_n = (int)ceil_div(r.N, kTileN);
        r.k_blocks = (int)ceil_div(r.K, kDepth), r.splits = splits[i];
        r.parts = r.splits > 1 || q.joins, r.part = b.part[i];
        r.ld = (int)round_up(r.N, 4);
        const int64_t e = 16 / (int64_t)esize;
        r.linear = r.V >= r.row0 + r.M;
        r.twos = esize == 2 && r.sc == 1 && ((uintptr_t)r.out & 3) == 0 && r.N % 2 == 0 && r.sm % 2 == 0 && r.sn % 2 == 0;
        r.vec = r.sc == 1 && ((uintptr_t)r.out & 15) == 0 && r.N % e == 0 && r.sm % e == 0 && r.sn % e == 0;
        if ((int64_t)r.tiles_m * r.tiles_n * r.splits > 0x7fffffff) MSD_FAIL(MSD_ERR_UNSUPPORTED, "linear cross entropy: %d x %d gradients are too many", r.M, r.N);
    }
    m.sum_blocks = kSumBack;
    assign(&m, pairs, dx != nullptr, dw != nullptr);
    XENT_TRY(launch_mma<kBack>(m, q.P, (dx && ceil_div(X.k_blocks, X.splits) > kSumBack) || (dw && ceil_div(W.k_blocks, W.splits) > kSumBack), pairs, s));
    for (int i = 0; i < 2; ++i)
        if (m.p[i].parts && (i == 0 ? dx != nullptr : dw != nullptr)) {
            join_kernel<<<(unsigned)ceil_div((int64_t)m.p[i].M * m.p[i].N, m.p[i].splits <= kFewSplits ? kThreads : 32), kThreads, 0, s>>>(m, i, p.dtype);
            XENT_TRY(launched());
        }
    return MSD_OK;
}

int backward(const Problem &p, const float *saved, const float *grad_loss, const Features *dx, void *dw, void *db, void *ws, size_t wsb, int device,
             cudaStream_t s) {
    if (narrow_supported(p) && (dx || dw || db)) return narrow_backward(p, nullptr, const_cast<float *>(saved), grad_loss, dx, dw, db, ws, wsb, device, s);
    const Plan q = make_plan(p, true);
    const size_t esize = p.dtype == MSD_F32 ? 4 : 2;
    if (q.T == 0) {
        if (dw) MSD_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)q.O * q.C * esize, s));
        if (db) MSD_CUDA_TRY(cudaMemsetAsync(db, 0, (size_t)q.O * esize, s));
        return MSD_OK;
    }
    if (!dx && !dw && !db) return MSD_OK;
    Carver c(ws);
    const BackwardSpace b = carve_backward(q, &c);
    if (!ws || wsb < c.used) MSD_FAIL(MSD_ERR_WORKSPACE, "linear cross entropy backward: workspace of %zu bytes needed, %zu given", c.used, wsb);
    const int sms = fast::sm_count(device), pairs = pair_count(sms);
    const bool kept = kept_by_forward(p, q), per_token = p.reduction == MSD_REDUCE_NONE;
    Carver k(kept ? (char *)const_cast<float *>(saved) + stats_bytes(q) : (char *)ws + c.used);
    const Operands op = carve_operands(q, &k);
    if (!kept) {
        if (wsb < c.used + k.used) MSD_FAIL(MSD_ERR_WORKSPACE, "linear cross entropy backward: workspace of %zu bytes needed, %zu given", c.used + k.used, wsb);
    }
    const Stats stats = Stats::of(const_cast<float *>(saved), q.T);
    const Factor factor = per_token ? Factor{nullptr, nullptr} : Factor{grad_loss, stats.factor};
    for (int64_t t0 = 0; t0 < q.T; t0 += q.chunk) {
        const int64_t T_ = q.T - t0 < q.chunk ? q.T - t0 : q.chunk;
        if (!kept) XENT_TRY(pack_operands(p, q, op, t0, T_, s));
        for (int64_t o0 = 0; o0 < q.O; o0 += q.width) XENT_TRY(backward_piece(p, q, op, b, stats, per_token ? grad_loss : nullptr, factor, t0, T_, o0, dx, dw, db, device, pairs, s));
    }
    return MSD_OK;
}

}  // namespace xent
}  // namespace msd

// ---- C entry points ----------------------------------------------------------------------
using namespace msd;

static int xent_problem(const char *op, int dtype, const msd_features_t *x, const void *weight, const void *bias, const int64_t *target, int64_t labels,
                        int64_t ignore_index, int reduction, xent::Problem *p) {
    if (dtype != MSD_F32 && dtype != MSD_BF16 && dtype != MSD_F16) MSD_FAIL(MSD_ERR_UNSUPPORTED, "%s: dtype %d is not MSD_F32, MSD_BF16 or MSD_F16", op, dtype);
    if (!x || x->batch < 0 || x->channels < 1 || x->voxels < 0) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: features need at least one channel and sizes of zero or more", op);
    if (labels < 1) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: at least one label is needed", op);
    if (reduction != MSD_REDUCE_NONE && reduction != MSD_REDUCE_MEAN && reduction != MSD_REDUCE_SUM)
        MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: reduction %d is not MSD_REDUCE_NONE, MSD_REDUCE_MEAN or MSD_REDUCE_SUM", op, reduction);
    const int64_t limit = ((int64_t)1 << 31) - 1024;  // whole tiles past the last row still count in 32 bits
    if (x->channels > (1 << 20) || labels >= limit) MSD_FAIL(MSD_ERR_UNSUPPORTED, "%s: at most 2^20 channels and 2^31 - 1024 labels", op);
    if (x->voxels && x->batch >= limit / x->voxels) MSD_FAIL(MSD_ERR_UNSUPPORTED, "%s: at most 2^31 - 1024 voxels", op);
    if (x->batch * x->voxels > 0 && (!x->data || !target)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: features and target must not be null", op);
    if (!weight) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "%s: weight must not be null", op);
    p->dtype = dtype;
    p->x = {x->data, x->batch, x->channels, x->voxels, x->stride_batch, x->stride_channel, x->stride_voxel};
    p->weight = weight, p->bias = bias, p->target = target;
    p->labels = labels, p->ignore_index = ignore_index, p->reduction = reduction;
    return MSD_OK;
}

static int xent_saved(const char *op, const xent::Problem &p, const void *saved, size_t bytes) {
    if ((uintptr_t)saved & 255) MSD_FAIL(MSD_ERR_WORKSPACE, "%s: saved must be 256-byte aligned", op);
    const size_t need = xent::saved_bytes(p);
    if (bytes < need) MSD_FAIL(MSD_ERR_WORKSPACE, "%s: %zu bytes to be saved, %zu given", op, need, bytes);
    return MSD_OK;
}

extern "C" MSD_API size_t msd_linear_xent_workspace_bytes(int dtype, const msd_features_t *x, const void *weight, int64_t labels, int backward) {
    xent::Problem p;
    msd_features_t f;
    if (!x) return 0;
    f = *x;
    f.data = (void *)(uintptr_t)256;
    if (xent_problem("msd_linear_xent_workspace_bytes", dtype, &f, weight, nullptr, (const int64_t *)f.data, labels, 0, MSD_REDUCE_MEAN, &p)) return 0;
    return backward ? xent::backward_workspace_bytes(p) : xent::forward_workspace_bytes(p);
}

extern "C" MSD_API size_t msd_linear_xent_saved_bytes(int dtype, const msd_features_t *x, const void *weight, int64_t labels) {
    xent::Problem p;
    msd_features_t f;
    if (!x) return 0;
    f = *x;
    f.data = (void *)(uintptr_t)256;
    if (xent_problem("msd_linear_xent_saved_bytes", dtype, &f, weight, nullptr, (const int64_t *)f.data, labels, 0, MSD_REDUCE_MEAN, &p)) return 0;
    return xent::saved_bytes(p);
}

extern "C" MSD_API int msd_linear_xent_single_pass(int dtype, const msd_features_t *x, int64_t labels) {
    xent::Problem p;
    msd_features_t f;
    if (!x) return 0;
    f = *x;
    f.data = (void *)(uintptr_t)256;
    if (xent_problem("msd_linear_xent_single_pass", dtype, &f, f.data, nullptr, (const int64_t *)f.data, labels, 0, MSD_REDUCE_MEAN, &p)) return 0;
    return xent::single_pass(p) ? 1 : 0;
}

extern "C" MSD_API int msd_linear_xent_forward(int dtype, const msd_features_t *x, const void *weight, const void *bias, const int64_t *target, int64_t labels,
                                               int64_t ignore_index, int reduction, float *loss, void *saved, size_t saved_bytes, void *workspace, size_t workspace_bytes,
                                               int device, void *stream) {
    xent::Problem p;
    int rc = xent_problem("msd_linear_xent_forward", dtype, x, weight, bias, target, labels, ignore_index, reduction, &p);
    if (rc) return rc;
    if (!loss && (reduction != MSD_REDUCE_NONE || p.x.tokens() > 0)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "msd_linear_xent_forward: loss must not be null");
    if (saved && (rc = xent_saved("msd_linear_xent_forward", p, saved, saved_bytes))) return rc;
    if (workspace && ((uintptr_t)workspace & 255)) MSD_FAIL(MSD_ERR_WORKSPACE, "msd_linear_xent_forward: workspace must be 256-byte aligned");
    DeviceGuard g(device);
    MSD_CUDA_TRY(g.status);
    return xent::forward(p, loss, (float *)saved, workspace, workspace_bytes, device, (cudaStream_t)stream);
}

extern "C" MSD_API int msd_linear_xent_backward(int dtype, const msd_features_t *x, const void *weight, const void *bias, const int64_t *target, int64_t labels,
                                                int64_t ignore_index, int reduction, const void *saved, size_t saved_bytes, const float *grad_loss,
                                                const msd_features_t *grad_x, void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes,
                                                int device, void *stream) {
    xent::Problem p;
    int rc = xent_problem("msd_linear_xent_backward", dtype, x, weight, bias, target, labels, ignore_index, reduction, &p);
    if (rc) return rc;
    if (!saved || (!grad_loss && p.x.tokens() > 0)) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "msd_linear_xent_backward: saved and grad_loss must not be null");
    if ((rc = xent_saved("msd_linear_xent_backward", p, saved, saved_bytes))) return rc;
    if (workspace && ((uintptr_t)workspace & 255)) MSD_FAIL(MSD_ERR_WORKSPACE, "msd_linear_xent_backward: workspace must be 256-byte aligned");
    xent::Features dx{};
    if (grad_x) {
        if (grad_x->batch != x->batch || grad_x->channels != x->channels || grad_x->voxels != x->voxels || (!grad_x->data && p.x.tokens() > 0))
            MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "msd_linear_xent_backward: grad_x differs in shape from the features");
        dx = {grad_x->data, grad_x->batch, grad_x->channels, grad_x->voxels, grad_x->stride_batch, grad_x->stride_channel, grad_x->stride_voxel};
    }
    DeviceGuard g(device);
    MSD_CUDA_TRY(g.status);
    return xent::backward(p, (const float *)saved, grad_loss, grad_x ? &dx : nullptr, grad_weight, grad_bias, workspace, workspace_bytes, device, (cudaStream_t)stream);
}

extern "C" MSD_API int msd_linear_xent_step(int dtype, const msd_features_t *x, const void *weight, const void *bias, const int64_t *target, int64_t labels,
                                            int64_t ignore_index, int reduction, float *loss, void *saved, size_t saved_bytes, const msd_features_t *grad_x, void *grad_weight,
                                            void *grad_bias, void *workspace, size_t workspace_bytes, int device, void *stream) {
    xent::Problem p;
    int rc = xent_problem("msd_linear_xent_step", dtype, x, weight, bias, target, labels, ignore_index, reduction, &p);
    if (rc) return rc;
    if (!loss || !saved) MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "msd_linear_xent_step: loss and saved must not be null");
    if ((rc = xent_saved("msd_linear_xent_step", p, saved, saved_bytes))) return rc;
    if (workspace && ((uintptr_t)workspace & 255)) MSD_FAIL(MSD_ERR_WORKSPACE, "msd_linear_xent_step: workspace must be 256-byte aligned");
    if (reduction == MSD_REDUCE_NONE || !xent::single_pass(p))
        MSD_FAIL(MSD_ERR_UNSUPPORTED, "msd_linear_xent_step: needs a mean or a sum, and a call that msd_linear_xent_single_pass accepts");
    xent::Features dx{};
    if (grad_x) {
        if (grad_x->batch != x->batch || grad_x->channels != x->channels || grad_x->voxels != x->voxels || !grad_x->data)
            MSD_FAIL(MSD_ERR_BAD_ARGUMENT, "msd_linear_xent_step: grad_x differs in shape from the features");
        dx = {grad_x->data, grad_x->batch, grad_x->channels, grad_x->voxels, grad_x->stride_batch, grad_x->stride_channel, grad_x->stride_voxel};
    }
    DeviceGuard g(device);
    MSD_CUDA_TRY(g.status);
    return xent::narrow_backward(p, loss, (float *)saved, nullptr, grad_x ? &dx : nullptr, grad_weight, grad_bias, workspace, workspace_bytes, device, (cudaStream_t)stream);
}
