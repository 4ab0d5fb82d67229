// Definitions shared by the causal attention kernels: the problem, its sequences, rows outside of them.
#pragma once

#include <cuda_runtime.h>

#include "sa_common.cuh"
#include "sa_host.cuh"

namespace sa {
namespace causal {

// Problem descriptor handed to every kernel by value.
struct CParams {
    int B, Nq, Nk, H, Hkv, D, G;         // G = H / Hkv query heads per KV head
    int S;                               // sequences; without cu_q those are the batch elements
    int max_q, max_k;                    // bounds of the lengths, for launch shapes only
    const int* cu_q;                     // NULL: every batch element is a sequence
    const int* cu_k;
    float scale;
    sa_strides q, k, v, o, d_o, dq, dk, dv;
};

// Columns of the tensor-core kernels' tiles: the head dim, filled up with zeros by the loads.
inline int tile_columns(int D) { return D <= 64 ? 64 : 128; }

// Rows of one sequence: queries [q0, q0 + nq) and keys [k0, k0 + nk) of batch element b.  Query i (from 0) sees keys
// j <= i + off, off = nk - nq.
struct Seq {
    int b, q0, nq, k0, nk;
    int id;                              // its number: of the batch element, or among the packed ones
    __device__ __forceinline__ int off() const { return nk - nq; }
};

// Whatever cu_q and cu_k hold, the rows are rows of the tensors.
__device__ __forceinline__ void clipped(const int* cu, int s, int n, int& start, int& len) {
    start = min(max(cu[s], 0), n);
    len = min(max(cu[s + 1], start), n) - start;
}
__device__ __forceinline__ Seq seq_of(const CParams& p, int s) {
    Seq r;
    r.id = s;
    if (p.cu_q == nullptr) {
        r.b = s;
        r.q0 = r.k0 = 0;
        r.nq = p.Nq;
        r.nk = p.Nk;
    } else {
        r.b = 0;
        clipped(p.cu_q, s, p.Nq, r.q0, r.nq);
        clipped(p.cu_k, s, p.Nk, r.k0, r.nk);
    }
    return r;
}

// Zeroes the rows of a packed tensor before the first and behind the last sequence (there are none as a rule: two loads).
// `block` of `blocks` equal shares, every thread of the block takes part.
template <typename T>
__device__ __forceinline__ void zero_outside(T* x, const sa_strides& st, int heads, int D, int n, const int* cu, int S, int block, int blocks) {
    const int first = min(max(cu[0], 0), n), last = max(min(max(cu[S], 0), n), first);
    const int out = first + n - last;
    for (int i = block; i < out; i += blocks) {
        T* row = x + (int64_t)(i < first ? i : last + i - first) * st.n;
        for (int e = threadIdx.x; e < heads * D; e += blockDim.x) row[(int64_t)(e / D) * st.h + e % D] = from_f<T>(0.f);
    }
}
__device__ __forceinline__ void empty_lse_outside(float* lse, int H, int n, const int* cu, int S, int block, int blocks) {
    const int first = min(max(cu[0], 0), n), last = max(min(max(cu[S], 0), n), first);
    const int out = first + n - last;
    for (int i = block; i < out; i += blocks)
        for (int h = threadIdx.x; h < H; h += blockDim.x) lse[(int64_t)h * n + (i < first ? i : last + i - first)] = -INFINITY;
}

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Estimated time of `units` walks, of `longest` steps at most and `mean` on average, each cut into `shares`, in steps: walks of
// different lengths, the longest first, end together; equal ones go by whole rounds over the multiprocessors.
inline double walk_steps(double units, int longest, double mean, int shares, int sms) {
    const int share = ceil_div(longest, shares);
    if (mean < 0.75 * longest) {
        const double all = units * mean / sms + 0.5;
        return all > share ? all : share;
    }
    return (double)(int64_t)((units * shares + sms - 1) / sms) * share;
}
// Steps on average: a causal prompt's queries see half of the keys.
inline double mean_steps(const CParams& c, int longest) { return c.max_q == c.max_k ? 0.5 * (longest + 1) : longest; }

// Shares of a walk: what makes the estimate least.  `joining` is what adding up shares costs, `each` what every share adds to
// that, in steps.
inline int plan_shares(double units, int longest, double mean, int sms, int most, double joining, double each) {
    int shares = 1;
    double best = walk_steps(units, longest, mean, 1, sms);
    for (int s = 2; s <= most && s <= longest && units * (s - 1) < 2.0 * sms; ++s) {
        const double cost = walk_steps(units, longest, mean, s, sms) + joining + each * s;
        if (cost < best) {
            best = cost;
            shares = s;
        }
    }
    return shares;
}

}  // namespace causal
}  // namespace sa
