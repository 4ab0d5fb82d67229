// Causal attention on the CUDA cores, fp32 arithmetic for every dtype, head dim (<= 256) and stride.  The on-device
// cross-check of the tensor-core kernels, and what fp32 tensors and other head dims take.
//
// A block of 16 x 16 threads works on tiles of 64 queries by 64 keys (32 keys above D = 128), staged in shared memory as
// fp32; a thread holds 4 rows by 4 (2) columns of the scores and 4 rows by D / 16 columns of the accumulators, so an operand
// read from shared memory is used four times.  Large problems are bound by the FMA pipes and shared-memory reads, small ones
// by the chain of loads, scores, softmax and products of a block.  Forward: one pass over the keys with the running maximum
// and sum of every row.  Backward: Delta = sum_d dO O once per row, then one kernel that owns queries (dQ) and one that owns
// keys and sums over the query heads of their KV head (dK, dV): no atomics, every sum in a fixed order.  Where a problem has
// fewer blocks than multiprocessors, a block's walk is cut into shares whose fp32 results are joined by a second kernel.
//
// Measured, fp32: B 1 N 256 H 2 D 64 forward 20 us, backward 42 us, with their joining kernels; bf16 B 2 N 8192 H 8 D 128, which the
// tensor-core kernels take otherwise, forward 13.6 ms (20 TFLOP/s).
//
// Scores outside the mask never enter an arithmetic operation: what NaN or infinity lies in keys a query does not see, or
// in rows of other sequences, does not reach it.
#pragma once

#include "sa_causal.cuh"

namespace sa {
namespace causal {

constexpr int kGenThreads = 256;
constexpr int kGenRows = 64;          // queries of a tile

template <int DP>
struct GenShape {
    static constexpr int kCols = DP <= 128 ? 64 : 32;      // keys of a tile
    static constexpr int kCpt = kCols / 16;                // score columns per thread, 16 apart
    static constexpr int kPitch = DP + 4;                  // floats: 16-byte reads of consecutive rows fall into different banks
    static constexpr int kPPitch = kCols + 4;
    static constexpr int kDpt = DP / 16;                   // accumulator columns per thread
    static constexpr int kVec = kDpt < 4 ? kDpt : 4;       // ... in groups of kVec consecutive ones, 16 kVec apart
    static constexpr int kRowTile = kGenRows * kPitch;
    static constexpr int kColTile = kCols * kPitch;
    static constexpr int kPTile = kGenRows * kPPitch;
    static constexpr int kFwdBytes = (kRowTile + 2 * kColTile + kPTile) * 4;
    static constexpr int kDqBytes = (2 * kRowTile + 2 * kColTile + kPTile) * 4;
    static constexpr int kDkvBytes = (2 * kRowTile + 2 * kColTile + 2 * kPTile) * 4;
    static_assert(kDkvBytes <= 227 * 1024 && kDqBytes <= 227 * 1024, "shared memory of a block");
};

template <int N>
__device__ __forceinline__ void lds_vec(const float* p, float (&v)[N]) {
    if constexpr (N == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else if constexpr (N == 2) {
        const float2 t = *reinterpret_cast<const float2*>(p);
        v[0] = t.x; v[1] = t.y;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = p[e];
    }
}

// Rows [r0, r0 + ROWS) of `x` (row stride sn, valid rows [0, n)) as fp32; rows and columns that do not exist are zeros.
template <typename T, int ROWS, int DP>
__device__ __forceinline__ void load_rows(float* tile, const T* x, int64_t sn, int r0, int n, int D) {
    constexpr int kPer = ROWS * DP / kGenThreads, kUnroll = kPer < 16 ? kPer : 16;
#pragma unroll 1
    for (int k0 = 0; k0 < kPer; k0 += kUnroll) {
        float v[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int e = threadIdx.x + (k0 + k) * kGenThreads, r = e / DP, d = e % DP;
            v[k] = r0 + r < n && d < D ? to_f<T>(x[(int64_t)(r0 + r) * sn + d]) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int e = threadIdx.x + (k0 + k) * kGenThreads;
            tile[e / DP * GenShape<DP>::kPitch + e % DP] = v[k];
        }
    }
}

// s[r][c] = A[4 ty + r] . B[tx + 16 c]
template <int DP>
__device__ __forceinline__ void dot_tile(const float* a, const float* b, int ty, int tx, float (&s)[4][GenShape<DP>::kCpt]) {
    using L = GenShape<DP>;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < L::kCpt; ++c) s[r][c] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float x[4][4], y[L::kCpt][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) lds_vec<4>(a + (4 * ty + r) * L::kPitch + d, x[r]);
#pragma unroll
        for (int c = 0; c < L::kCpt; ++c) lds_vec<4>(b + (tx + 16 * c) * L::kPitch + d, y[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < L::kCpt; ++c) s[r][c] = fmaf(x[r][e], y[c][e], s[r][c]);
    }
}

// acc[r][.] += sum_x w[r](x) * rows[x][.] over `count` rows; weight r of row x is w[x * sx + r * sr].  With MASKED a weight of
// zero skips the product (the row may be NaN or infinite where it is masked).
template <int DP, int R, bool MASKED>
__device__ __forceinline__ void accumulate(float (&acc)[R][GenShape<DP>::kDpt], const float* w, int sx, int sr, const float* rows, int count, int tx) {
    using L = GenShape<DP>;
#pragma unroll 4
    for (int x = 0; x < count; ++x) {
        float wv[R];
#pragma unroll
        for (int r = 0; r < R; ++r) wv[r] = w[x * sx + r * sr];
#pragma unroll
        for (int g = 0; g < L::kDpt / L::kVec; ++g) {
            float v[L::kVec];
            lds_vec<L::kVec>(rows + x * L::kPitch + 16 * L::kVec * g + L::kVec * tx, v);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < L::kVec; ++e) {
                    float& t = acc[r][g * L::kVec + e];
                    if (MASKED) t = wv[r] == 0.f ? t : fmaf(wv[r], v[e], t);
                    else t = fmaf(wv[r], v[e], t);
                }
        }
    }
}

// (with `low`: what rounding took, too)
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* row, const float (&v)[GenShape<DP>::kDpt], float f, int tx, int D, T* low = nullptr) {
    using L = GenShape<DP>;
#pragma unroll
    for (int g = 0; g < L::kDpt / L::kVec; ++g)
#pragma unroll
        for (int e = 0; e < L::kVec; ++e) {
            const int d = 16 * L::kVec * g + L::kVec * tx + e;
            if (d < D) {
                const float x = v[g * L::kVec + e] * f;
                const T t = from_f<T>(x);
                row[d] = t;
                if (low) low[d] = from_f<T>(x - to_f<T>(t));
            }
        }
}

// A block's place: its rows (or keys), head and sequence, share.
struct GenPlace {
    int blk, h, s, share;
    bool first;              // of the blocks that share the rows outside the sequences
    __device__ __forceinline__ GenPlace(int heads, int S, int shares) {
        int x = blockIdx.x;
        share = x % shares;
        x /= shares;
        first = share == 0 && x % (heads * S) == 0;
        h = x % heads;
        x /= heads;
        s = x % S;
        blk = x / S;
    }
};

__device__ __forceinline__ float half_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kGenThreads) causal_fwd_kernel(const CParams p, const T* __restrict__ q, const T* __restrict__ k,
                                                                const T* __restrict__ v, T* __restrict__ o, T* __restrict__ o_low, float* __restrict__ lse,
                                                                int blocks_q, int shares, float* __restrict__ part_o, float* __restrict__ part_lse) {
    using L = GenShape<DP>;
    extern __shared__ float4 smem4[];
    float* const qt = reinterpret_cast<float*>(smem4);
    float* const kt = qt + L::kRowTile;
    float* const vt = kt + L::kColTile;
    float* const pt = vt + L::kColTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    // the longest rows first: the last blocks to start are the short ones
    const GenPlace at(p.H, p.S, shares);
    const int blk = blocks_q - 1 - at.blk, h = at.h;
    const Seq s = seq_of(p, at.s);
    const int64_t rows = (int64_t)p.B * p.H * p.Nq, row0 = ((int64_t)s.b * p.H + h) * p.Nq + s.q0;
    q += s.b * p.q.b + s.q0 * p.q.n + h * p.q.h;
    k += s.b * p.k.b + s.k0 * p.k.n + h / p.G * p.k.h;
    v += s.b * p.v.b + s.k0 * p.v.n + h / p.G * p.v.h;
    o += s.b * p.o.b + s.q0 * p.o.n + h * p.o.h;
    if (o_low) o_low += s.b * p.o.b + s.q0 * p.o.n + h * p.o.h;
    lse += ((int64_t)s.b * p.H + h) * p.Nq + s.q0;

    for (int i0 = blk * kGenRows; i0 < s.nq; i0 += blocks_q * kGenRows) {
        __syncthreads();
        load_rows<T, kGenRows, DP>(qt, q, p.q.n, i0, s.nq, p.D);
        float acc[4][L::kDpt], m[4], l[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int e = 0; e < L::kDpt; ++e) acc[r][e] = 0.f;
        }
        const int seen = max(min(i0 + kGenRows, s.nq) + s.off(), 0);        // keys the last row sees
        const int per = (ceil_div(seen, L::kCols) + shares - 1) / shares * L::kCols, j_begin = min(at.share * per, seen), j_end = min(j_begin + per, seen);
        for (int j0 = j_begin; j0 < j_end; j0 += L::kCols) {
            __syncthreads();
            load_rows<T, L::kCols, DP>(kt, k, p.k.n, j0, s.nk, p.D);
            load_rows<T, L::kCols, DP>(vt, v, p.v.n, j0, s.nk, p.D);
            __syncthreads();
            float x[4][L::kCpt];
            dot_tile<DP>(qt, kt, ty, tx, x);
            const bool masked = j0 + L::kCols - 1 > i0 + s.off();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int hi = i0 + 4 * ty + r + s.off() - j0;
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < L::kCpt; ++c) {
                    x[r][c] = tx + 16 * c <= hi ? x[r][c] * p.scale : -INFINITY;
                    top = fmaxf(top, x[r][c]);
                }
                const float mn = fmaxf(m[r], half_max(top)), base = mn == -INFINITY ? 0.f : mn;
                const float f = expf(m[r] - base);
                m[r] = mn;
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < L::kCpt; ++c) {
                    const float e = expf(x[r][c] - base);
                    sum += e;
                    pt[(4 * ty + r) * L::kPPitch + tx + 16 * c] = e;
                }
                l[r] = l[r] * f + sum;
#pragma unroll
                for (int e = 0; e < L::kDpt; ++e) acc[r][e] *= f;
            }
            __syncwarp();          // a row of P is written and read by the same half warp
            if (masked) accumulate<DP, 4, true>(acc, pt + 4 * ty * L::kPPitch, 1, L::kPPitch, vt, L::kCols, tx);
            else accumulate<DP, 4, false>(acc, pt + 4 * ty * L::kPPitch, 1, L::kPPitch, vt, L::kCols, tx);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 4 * ty + r;
            const float sum = half_sum(l[r]);
            if (i < s.nq) {
                const bool none = min(i + s.off(), j_end - 1) < j_begin || sum == 0.f;        // (or all scores are -inf)
                const float ll = none ? -INFINITY : m[r] + logf(sum);
                if (shares > 1) {
                    if (!none) store_row<float, DP>(part_o + (at.share * rows + row0 + i) * DP, acc[r], 1.f / sum, tx, p.D);
                    if (tx == 0) part_lse[at.share * rows + row0 + i] = ll;
                    continue;
                }
                store_row<T, DP>(o + (int64_t)i * p.o.n, acc[r], none ? 0.f : 1.f / sum, tx, p.D, o_low ? o_low + (int64_t)i * p.o.n : nullptr);
                if (tx == 0) lse[i] = ll;
            }
        }
    }
    if (p.cu_q != nullptr && at.first) {
        zero_outside(o - s.q0 * p.o.n - h * p.o.h, p.o, p.H, p.D, p.Nq, p.cu_q, p.S, blk, blocks_q);
        empty_lse_outside(lse - ((int64_t)h * p.Nq + s.q0), p.H, p.Nq, p.cu_q, p.S, blk, blocks_q);
    }
}

// Delta = sum_d dO O of every row, a warp per row and head.
template <typename T>
__global__ void __launch_bounds__(256) causal_delta_kernel(const CParams p, const T* __restrict__ o, const T* __restrict__ o_low, const T* __restrict__ d_o,
                                                          float* __restrict__ delta) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (int64_t)p.B * p.Nq * p.H) return;
    const int h = (int)(w % p.H), i = (int)(w / p.H % p.Nq), b = (int)(w / p.H / p.Nq);
    const int64_t at = b * p.o.b + i * p.o.n + h * p.o.h;
    d_o += b * p.d_o.b + i * p.d_o.n + h * p.d_o.h;
    float sum = 0.f;
    for (int d = lane; d < p.D; d += 32) sum = fmaf(to_f<T>(o[at + d]) + (o_low ? to_f<T>(o_low[at + d]) : 0.f), to_f<T>(d_o[d]), sum);
    sum = warp_sum(sum);
    if (lane == 0) delta[((int64_t)b * p.H + h) * p.Nq + i] = sum;
}

// The LSE that a row's scores are taken from: with that of a row whose scores are all -inf every P is zero, as in the forward.
__device__ __forceinline__ float lse_of_weights(float lse) { return lse == -INFINITY ? INFINITY : lse; }

// P and dS of a tile of queries i0.. and keys j0..: zero outside the mask.  (exp of a score against the row's LSE: a row that
// sees no key has no score inside the mask.)
template <int DP>
__device__ __forceinline__ void p_and_ds(const float (&x)[4][GenShape<DP>::kCpt], const float (&y)[4][GenShape<DP>::kCpt], const float (&ls)[4],
                                         const float (&dl)[4], int i0, int j0, const Seq& s, float scale, int ty, int tx, float* pt, float* dst) {
    using L = GenShape<DP>;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * ty + r, hi = i < s.nq ? min(i + s.off(), s.nk - 1) - j0 : -1;
#pragma unroll
        for (int c = 0; c < L::kCpt; ++c) {
            const bool in = tx + 16 * c <= hi;
            const float e = in ? expf(x[r][c] * scale - ls[r]) : 0.f;
            const int at = (4 * ty + r) * L::kPPitch + tx + 16 * c;
            if (pt) pt[at] = e;
            dst[at] = in ? e * (y[r][c] - dl[r]) * scale : 0.f;
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kGenThreads) causal_dq_kernel(const CParams p, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                               const float* __restrict__ lse, const float* __restrict__ delta, const T* __restrict__ d_o,
                                                               T* __restrict__ dq, int blocks_q, int shares, float* __restrict__ part) {
    using L = GenShape<DP>;
    extern __shared__ float4 smem4[];
    float* const qt = reinterpret_cast<float*>(smem4);
    float* const dt = qt + L::kRowTile;
    float* const kt = dt + L::kRowTile;
    float* const vt = kt + L::kColTile;
    float* const st = vt + L::kColTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const GenPlace at(p.H, p.S, shares);
    const int blk = blocks_q - 1 - at.blk, h = at.h;
    const Seq s = seq_of(p, at.s);
    const int64_t rows = (int64_t)p.B * p.H * p.Nq, row0 = ((int64_t)s.b * p.H + h) * p.Nq + s.q0;
    q += s.b * p.q.b + s.q0 * p.q.n + h * p.q.h;
    k += s.b * p.k.b + s.k0 * p.k.n + h / p.G * p.k.h;
    v += s.b * p.v.b + s.k0 * p.v.n + h / p.G * p.v.h;
    d_o += s.b * p.d_o.b + s.q0 * p.d_o.n + h * p.d_o.h;
    dq += s.b * p.dq.b + s.q0 * p.dq.n + h * p.dq.h;
    lse += ((int64_t)s.b * p.H + h) * p.Nq + s.q0;
    delta += ((int64_t)s.b * p.H + h) * p.Nq + s.q0;
    for (int i0 = blk * kGenRows; i0 < s.nq; i0 += blocks_q * kGenRows) {
        __syncthreads();
        load_rows<T, kGenRows, DP>(qt, q, p.q.n, i0, s.nq, p.D);
        load_rows<T, kGenRows, DP>(dt, d_o, p.d_o.n, i0, s.nq, p.D);
        float acc[4][L::kDpt], ls[4], dl[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 4 * ty + r;
            ls[r] = i < s.nq ? lse_of_weights(lse[i]) : 0.f;
            dl[r] = i < s.nq ? delta[i] : 0.f;
#pragma unroll
            for (int e = 0; e < L::kDpt; ++e) acc[r][e] = 0.f;
        }
        const int seen = max(min(i0 + kGenRows, s.nq) + s.off(), 0);
        const int per = (ceil_div(seen, L::kCols) + shares - 1) / shares * L::kCols, j_begin = min(at.share * per, seen), j_end = min(j_begin + per, seen);
        for (int j0 = j_begin; j0 < j_end; j0 += L::kCols) {
            __syncthreads();
            load_rows<T, L::kCols, DP>(kt, k, p.k.n, j0, s.nk, p.D);
            load_rows<T, L::kCols, DP>(vt, v, p.v.n, j0, s.nk, p.D);
            __syncthreads();
            float x[4][L::kCpt], y[4][L::kCpt];
            dot_tile<DP>(qt, kt, ty, tx, x);
            dot_tile<DP>(dt, vt, ty, tx, y);
            p_and_ds<DP>(x, y, ls, dl, i0, j0, s, p.scale, ty, tx, nullptr, st);
            __syncwarp();
            if (j0 + L::kCols - 1 > i0 + s.off()) accumulate<DP, 4, true>(acc, st + 4 * ty * L::kPPitch, 1, L::kPPitch, kt, L::kCols, tx);
            else accumulate<DP, 4, false>(acc, st + 4 * ty * L::kPPitch, 1, L::kPPitch, kt, L::kCols, tx);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (i0 + 4 * ty + r < s.nq) {
                if (shares > 1) store_row<float, DP>(part + (at.share * rows + row0 + i0 + 4 * ty + r) * DP, acc[r], 1.f, tx, p.D);
                else store_row<T, DP>(dq + (int64_t)(i0 + 4 * ty + r) * p.dq.n, acc[r], 1.f, tx, p.D);
            }
    }
    if (p.cu_q != nullptr && at.first) zero_outside(dq - s.q0 * p.dq.n - h * p.dq.h, p.dq, p.H, p.D, p.Nq, p.cu_q, p.S, blk, blocks_q);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kGenThreads) causal_dkv_kernel(const CParams p, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                                const float* __restrict__ lse, const float* __restrict__ delta, const T* __restrict__ d_o,
                                                                T* __restrict__ dk, T* __restrict__ dv, int blocks_k, int shares, float* __restrict__ part_k,
                                                                float* __restrict__ part_v) {
    using L = GenShape<DP>;
    constexpr int kOwn = L::kCols / 16;          // keys per thread
    extern __shared__ float4 smem4[];
    float* const qt = reinterpret_cast<float*>(smem4);
    float* const dt = qt + L::kRowTile;
    float* const kt = dt + L::kRowTile;
    float* const vt = kt + L::kColTile;
    float* const pt = vt + L::kColTile;
    float* const st = pt + L::kPTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    // the first keys are seen by the most queries: they go first
    const GenPlace at(p.Hkv, p.S, shares);
    const int blk = at.blk, hk = at.h;
    const Seq s = seq_of(p, at.s);
    const int64_t key0 = (((int64_t)at.share * p.B + s.b) * p.Hkv + hk) * p.Nk + s.k0;
    k += s.b * p.k.b + s.k0 * p.k.n + hk * p.k.h;
    v += s.b * p.v.b + s.k0 * p.v.n + hk * p.v.h;
    for (int j0 = blk * L::kCols; j0 < s.nk; j0 += blocks_k * L::kCols) {
        __syncthreads();
        load_rows<T, L::kCols, DP>(kt, k, p.k.n, j0, s.nk, p.D);
        load_rows<T, L::kCols, DP>(vt, v, p.v.n, j0, s.nk, p.D);
        float ak[kOwn][L::kDpt], av[kOwn][L::kDpt];
#pragma unroll
        for (int r = 0; r < kOwn; ++r)
#pragma unroll
            for (int e = 0; e < L::kDpt; ++e) ak[r][e] = av[r][e] = 0.f;
        const int i_first = max(j0 - s.off(), 0) / kGenRows * kGenRows;
        // steps of (query head of the group, query tile), this share's
        const int tiles = max(ceil_div(s.nq - i_first, kGenRows), 0), total = tiles * p.G, per = (total + shares - 1) / shares;
        const int it_end = min((at.share + 1) * per, total);
        for (int it = at.share * per; it < it_end; ++it) {
            const int h = hk * p.G + it / tiles, i0 = i_first + it % tiles * kGenRows;
            const T* qh = q + s.b * p.q.b + s.q0 * p.q.n + h * p.q.h;
            const T* dh = d_o + s.b * p.d_o.b + s.q0 * p.d_o.n + h * p.d_o.h;
            const int64_t row = ((int64_t)s.b * p.H + h) * p.Nq + s.q0;
            __syncthreads();
            load_rows<T, kGenRows, DP>(qt, qh, p.q.n, i0, s.nq, p.D);
            load_rows<T, kGenRows, DP>(dt, dh, p.d_o.n, i0, s.nq, p.D);
            float ls[4], dl[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = i0 + 4 * ty + r;
                ls[r] = i < s.nq ? lse_of_weights(lse[row + i]) : 0.f;
                dl[r] = i < s.nq ? delta[row + i] : 0.f;
            }
            __syncthreads();
            float x[4][L::kCpt], y[4][L::kCpt];
            dot_tile<DP>(qt, kt, ty, tx, x);
            dot_tile<DP>(dt, vt, ty, tx, y);
            p_and_ds<DP>(x, y, ls, dl, i0, j0, s, p.scale, ty, tx, pt, st);
            __syncthreads();
            const bool masked = j0 + L::kCols - 1 > i0 + s.off() || i0 + kGenRows > s.nq;
            if (masked) {
                accumulate<DP, kOwn, true>(av, pt + kOwn * ty, L::kPPitch, 1, dt, kGenRows, tx);
                accumulate<DP, kOwn, true>(ak, st + kOwn * ty, L::kPPitch, 1, qt, kGenRows, tx);
            } else {
                accumulate<DP, kOwn, false>(av, pt + kOwn * ty, L::kPPitch, 1, dt, kGenRows, tx);
                accumulate<DP, kOwn, false>(ak, st + kOwn * ty, L::kPPitch, 1, qt, kGenRows, tx);
            }
        }
#pragma unroll
        for (int r = 0; r < kOwn; ++r) {
            const int j = j0 + kOwn * ty + r;
            if (j < s.nk && shares > 1) {
                if (dk) store_row<float, DP>(part_k + (key0 + j) * DP, ak[r], 1.f, tx, p.D);
                if (dv) store_row<float, DP>(part_v + (key0 + j) * DP, av[r], 1.f, tx, p.D);
            } else if (j < s.nk) {
                if (dk) store_row<T, DP>(dk + s.b * p.dk.b + (int64_t)(s.k0 + j) * p.dk.n + hk * p.dk.h, ak[r], 1.f, tx, p.D);
                if (dv) store_row<T, DP>(dv + s.b * p.dv.b + (int64_t)(s.k0 + j) * p.dv.n + hk * p.dv.h, av[r], 1.f, tx, p.D);
            }
        }
    }
    if (p.cu_k != nullptr && at.first) {
        if (dk) zero_outside(dk, p.dk, p.Hkv, p.D, p.Nk, p.cu_k, p.S, blk, blocks_k);
        if (dv) zero_outside(dv, p.dv, p.Hkv, p.D, p.Nk, p.cu_k, p.S, blk, blocks_k);
    }
}

// Joins the shares of a row, a warp per row and head (see causal_join_kernel).
template <typename T, int DP>
__global__ void __launch_bounds__(256) causal_general_join_kernel(const CParams p, int shares, const float* __restrict__ part_o,
                                                                 const float* __restrict__ part_lse, T* __restrict__ o, T* __restrict__ o_low,
                                                                 float* __restrict__ lse) {
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)p.B * p.H * p.Nq, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (at >= rows) return;
    const int n = (int)(at % p.Nq), h = (int)(at / p.Nq % p.H), b = (int)(at / p.Nq / p.H);
    if (p.cu_q != nullptr && (n < p.cu_q[0] || n >= p.cu_q[p.S])) return;       // (written where the shares are)
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < shares; ++s) top = fmaxf(top, part_lse[s * rows + at]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int s = 0; s < shares; ++s) sum += expf(part_lse[s * rows + at] - base);
    const int64_t dst = b * p.o.b + (int64_t)n * p.o.n + h * p.o.h;
    for (int d = lane; d < p.D; d += 32) {
        float acc = 0.f;
        for (int s = 0; s < shares; ++s) {
            const float ls = part_lse[s * rows + at];
            if (ls != -INFINITY) acc = fmaf(expf(ls - base), part_o[(s * rows + at) * DP + d], acc);
        }
        acc = sum == 0.f ? 0.f : acc / sum;
        const T t = from_f<T>(acc);
        o[dst + d] = t;
        if (o_low) o_low[dst + d] = from_f<T>(acc - to_f<T>(t));
    }
    if (lane == 0) lse[at] = sum == 0.f ? -INFINITY : top + logf(sum);
}

// Adds the shares of a gradient in their order, a thread per element.
template <typename T, int DP>
__global__ void __launch_bounds__(256) causal_general_add_kernel(const float* __restrict__ part, T* __restrict__ out, sa_strides so, int shares, int B,
                                                                int heads, int n, int D, const int* cu, int S) {
    const int64_t rows = (int64_t)B * heads * n, idx = (int64_t)blockIdx.x * 256 + threadIdx.x, at = idx / D;
    if (at >= rows) return;
    const int d = (int)(idx - at * D), i = (int)(at % n), h = (int)(at / n % heads), b = (int)(at / n / heads);
    float sum = 0.f;
    if (cu == nullptr || (i >= cu[0] && i < cu[S]))           // (rows outside every sequence: zeros)
        for (int s = 0; s < shares; ++s) sum += part[(s * rows + at) * DP + d];
    out[b * so.b + (int64_t)i * so.n + h * so.h + d] = from_f<T>(sum);
}

// How a call is cut up, and its workspace.
struct GenPlan {
    int shares_q, shares_k;           // of a query tile's keys (forward, dQ), and of a key tile's steps
    size_t delta, part0, part1, part2, bytes;
};
inline GenPlan plan_general(const CParams& c, bool backward) {
    GenPlan f{};
    const int dp = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256, cols = dp <= 128 ? 64 : 32, sms = host::sm_count();
    // (a step takes about 4 us, joining 4)
    const int steps_q = ceil_div(c.max_k, cols), tiles = ceil_div(c.max_q, kGenRows), steps_k = (int)((int64_t)tiles * c.G < (1 << 20) ? tiles * c.G : 1 << 20);
    f.shares_q = plan_shares((double)tiles * c.H * c.S, steps_q, mean_steps(c, steps_q), sms, 16, 1, 0.05);
    f.shares_k = plan_shares((double)ceil_div(c.max_k, cols) * c.Hkv * c.S, steps_k, c.max_q == c.max_k ? 0.5 * steps_k : steps_k, sms, 16, 1, 0.05);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t x = at; at += (n + 255) / 256 * 256; return x; };
    const size_t rows = (size_t)c.B * c.H * c.Nq, keys = (size_t)c.B * c.Hkv * c.Nk;
    if (backward) {
        f.delta = take(rows * 4);
        f.part0 = take(f.shares_q > 1 ? f.shares_q * rows * dp * 4 : 0);
        f.part1 = take(f.shares_k > 1 ? f.shares_k * keys * dp * 4 : 0);
        f.part2 = take(f.shares_k > 1 ? f.shares_k * keys * dp * 4 : 0);
    } else {
        f.part0 = take(f.shares_q > 1 ? f.shares_q * rows * dp * 4 : 0);
        f.part1 = take(f.shares_q > 1 ? f.shares_q * rows * 4 : 0);
    }
    f.bytes = at;
    return f;
}

template <typename T, int DP>
int launch_general_fwd_d(const CParams& p, const void* q, const void* k, const void* v, void* o, void* o_low, float* lse, uint8_t* ws, cudaStream_t st) {
    using L = GenShape<DP>;
    const GenPlan f = plan_general(p, false);
    const int bq = ceil_div(p.max_q, kGenRows);
    const int64_t grid = (int64_t)bq * p.H * p.S * f.shares_q, rows = (int64_t)p.B * p.H * p.Nq;
    if (grid > 0x7fffffff || rows > 0x7fffffff) return SA_ERR_UNSUPPORTED;
    auto kern = causal_fwd_kernel<T, DP>;
    if (!allow_dynamic_smem((const void*)kern, L::kFwdBytes)) return SA_ERR_LAUNCH;
    float *po = reinterpret_cast<float*>(ws + f.part0), *pl = reinterpret_cast<float*>(ws + f.part1);
    kern<<<(unsigned)grid, kGenThreads, L::kFwdBytes, st>>>(p, (const T*)q, (const T*)k, (const T*)v, (T*)o, (T*)o_low, lse, bq, f.shares_q, po, pl);
    host::count_launches(1);
    if (f.shares_q > 1) {
        causal_general_join_kernel<T, DP><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p, f.shares_q, po, pl, (T*)o, (T*)o_low, lse);
        host::count_launches(1);
    }
    return cudaGetLastError() == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
}

template <typename T, int DP>
int launch_general_bwd_d(const CParams& p, const void* q, const void* k, const void* v, const void* o, const void* o_low, const float* lse, const void* d_o,
                         void* dq, void* dk, void* dv, uint8_t* ws, cudaStream_t st) {
    using L = GenShape<DP>;
    const GenPlan f = plan_general(p, true);
    const int bq = ceil_div(p.max_q, kGenRows), bk = ceil_div(p.max_k, L::kCols);
    const int64_t gq = (int64_t)bq * p.H * p.S * f.shares_q, gk = (int64_t)bk * p.Hkv * p.S * f.shares_k, rows = (int64_t)p.B * p.Nq * p.H;
    if (gq > 0x7fffffff || gk > 0x7fffffff || rows > 0x7fffffff) return SA_ERR_UNSUPPORTED;
    if (!allow_dynamic_smem((const void*)causal_dq_kernel<T, DP>, L::kDqBytes) || !allow_dynamic_smem((const void*)causal_dkv_kernel<T, DP>, L::kDkvBytes))
        return SA_ERR_LAUNCH;
    float* delta = reinterpret_cast<float*>(ws + f.delta);
    causal_delta_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p, (const T*)o, (const T*)o_low, (const T*)d_o, delta);
    host::count_launches(1);
    auto add = [&](const float* part, void* out, const sa_strides& so, int shares, int heads, int n, const int* cu) {
        const int64_t all = (int64_t)p.B * heads * n * p.D;
        causal_general_add_kernel<T, DP><<<(unsigned)((all + 255) / 256), 256, 0, st>>>(part, (T*)out, so, shares, p.B, heads, n, p.D, cu, p.S);
        host::count_launches(1);
    };
    if (dq) {
        float* part = reinterpret_cast<float*>(ws + f.part0);
        causal_dq_kernel<T, DP><<<(unsigned)gq, kGenThreads, L::kDqBytes, st>>>(p, (const T*)q, (const T*)k, (const T*)v, lse, delta, (const T*)d_o, (T*)dq, bq,
                                                                                f.shares_q, part);
        host::count_launches(1);
        if (f.shares_q > 1) add(part, dq, p.dq, f.shares_q, p.H, p.Nq, p.cu_q);
    }
    if (dk || dv) {
        float *pk = reinterpret_cast<float*>(ws + f.part1), *pv = reinterpret_cast<float*>(ws + f.part2);
        causal_dkv_kernel<T, DP><<<(unsigned)gk, kGenThreads, L::kDkvBytes, st>>>(p, (const T*)q, (const T*)k, (const T*)v, lse, delta, (const T*)d_o, (T*)dk, (T*)dv,
                                                                                  bk, f.shares_k, pk, pv);
        host::count_launches(1);
        if (f.shares_k > 1 && dk) add(pk, dk, p.dk, f.shares_k, p.Hkv, p.Nk, p.cu_k);
        if (f.shares_k > 1 && dv) add(pv, dv, p.dv, f.shares_k, p.Hkv, p.Nk, p.cu_k);
    }
    return cudaGetLastError() == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
}

// f(element type, head dim rounded up to what is instantiated)
template <typename F>
int dispatch_general(int dtype, int D, F&& f) {
    auto by_d = [&](auto t) {
        if (D <= 64) return f(t, std::integral_constant<int, 64>{});
        if (D <= 128) return f(t, std::integral_constant<int, 128>{});
        return f(t, std::integral_constant<int, 256>{});
    };
    if (dtype == SA_BF16) return by_d(__nv_bfloat16{});
    if (dtype == SA_F16) return by_d(__half{});
    return by_d(float{});
}

}  // namespace causal
}  // namespace sa
