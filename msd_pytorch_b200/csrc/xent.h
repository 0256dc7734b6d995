// Internal interface of the linear layer with softmax cross entropy behind it (xent*.cu).
//
//   z[t,o]  = b[o] + sum_c x[t,c] W[o,c]          t = token (voxel), o = label, c = channel
//   lse[t]  = log sum_o exp z[t,o]
//   loss[t] = lse[t] - z[t,y_t]                   0 where y_t == ignore_index
//   G[t,o]  = g_t (exp(z[t,o] - lse[t]) - [o == y_t])
//   dx = G W,  dW = G^T x,  db[o] = sum_t G[t,o]
//
// The logits are never stored: forward keeps lse (7 bytes per token), backward computes them
// again.
//
// lse = m + log s with m the largest logit and s the sum of exp(z - m) >= 1.  Where a token is confident,
// loss and 1 - p are as small as log s while m is of the logits' size: lse rounded to a float would leave
// nothing of them (two logits near 100 and 11 apart: 27 % off).  So the target's logit is taken off m before
// log s is added, and backward gets lse in 48 bits: its float, and what that leaves in 24 bits.
// Logits are multiplied by log2(e) (the exponential's base is 2) once the maximum is off: a mask of the
// type's lowest value would leave the range.
#pragma once
#include "common.cuh"

namespace msd {
namespace xent {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Features {  // x or dx: element (n, c, v) at data[n*sn + c*sc + v*sv]; token = n*V + v
    void *p;
    int64_t N, C, V;
    int64_t sn, sc, sv;
    int64_t tokens() const { return N * V; }
};

// log-sum-exps of T tokens and the factor of the reduction, in one buffer.
struct Stats {
    float *lse, *factor;
    uint16_t *low;  // the rest in units of 2^-24 of lse's last place (which counts as 64 at most: the rest of
    int8_t *high;   // m + log s is never more than log s <= 22): 16 bits and 8 bits of an integer
    static __host__ __device__ size_t lse_bytes(int64_t T) { return ((size_t)(T + 1) * sizeof(float) + 255) / 256 * 256; }
    static size_t bytes(int64_t T) { return lse_bytes(T) + ((size_t)T * 3 + 255) / 256 * 256; }
    static __host__ __device__ Stats of(void *base, int64_t T) {
        Stats s{(float *)base, nullptr, nullptr, nullptr};
        if (!base) return s;
        s.factor = s.lse + T;
        s.low = (uint16_t *)((char *)base + lse_bytes(T));
        s.high = (int8_t *)(s.low + T);
        return s;
    }
    __host__ __device__ Stats at(int64_t t) const { return lse ? Stats{lse + t, factor, low + t, high + t} : *this; }
#ifdef __CUDACC__
    static __device__ __forceinline__ float unit(float v) {
        const int e = (int)(__float_as_uint(v) >> 23 & 255);
        return __uint_as_float((uint32_t)(min(max(e, 48), 156) - 47) << 23);
    }
    __device__ __forceinline__ void write(int64_t t, float m, float log_s) const {
        const float sum = m + log_s, back = sum - m;
        const float rest = (m - (sum - back)) + (log_s - back);  // m + log_s = sum + rest
        const int code = fabsf(sum) < __uint_as_float(0x7f800000u) ? min((int)rintf(rest / unit(sum)), (1 << 23) - 1) : 0;
        lse[t] = sum, low[t] = (uint16_t)code, high[t] = (int8_t)(code >> 16);
    }
    __device__ __forceinline__ void read(int64_t t, float &sum, float &rest) const {
        sum = lse[t];
        rest = (float)((int)high[t] * 65536 + (int)low[t]) * unit(sum);
    }
#endif
};

struct Problem {
    int dtype;  // MSD_F32, MSD_BF16 or MSD_F16: x, W, b and their gradients
    Features x;
    const void *weight;     // [O][C] dense
    const void *bias;       // [O] or null
    const int64_t *target;  // [tokens]
    int64_t labels, ignore_index;
    int reduction;
};

// Few labels over voxels that lie side by side (xent_narrow.cu): loss and gradients can be had in
// one pass over x.
bool narrow_supported(const Problem &p);
bool single_pass(const Problem &p);
size_t narrow_workspace_bytes(const Problem &p);
// stats: one float, the factor of the reduction
int narrow_forward(const Problem &p, float *loss, float *stats, void *ws, size_t wsb, int device, cudaStream_t s);
// loss non-null: writes it too (mean or sum) and takes the upstream gradient as 1
int narrow_backward(const Problem &p, float *loss, float *stats, const float *grad_loss, const Features *dx, void *dw, void *db, void *ws, size_t wsb,
                    int device, cudaStream_t s);

// `saved`: what forward leaves to backward (its layout is the library's), or null without gradients.
size_t forward_workspace_bytes(const Problem &p);
size_t backward_workspace_bytes(const Problem &p);
size_t saved_bytes(const Problem &p);
int forward(const Problem &p, float *loss, float *saved, void *ws, size_t wsb, int device, cudaStream_t s);
int backward(const Problem &p, const float *saved, const float *grad_loss, const Features *dx, void *dw, void *db, void *ws, size_t wsb, int device,
             cudaStream_t s);

}  // namespace xent
}  // namespace msd
