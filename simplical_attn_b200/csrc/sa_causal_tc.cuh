// What the tensor-core causal attention kernels share: units of work, their order, the plan of a packed batch.
#pragma once

#include "sa_causal.cuh"
#include "sa_ptx.cuh"

namespace sa {
namespace causal {

constexpr int kTile = 128;            // rows of a query tile = lanes of tensor memory, and keys of a key tile

// 2^x of two values on the FMA pipes, for x up to 100: x = n + f with n whole and |f| <= 1/2, 2^f by a polynomial of degree 4
// (minimax of the relative error, 2.7e-6, fitted by reweighted least squares at Chebyshev points), 2^n from the bits of n.  Below
// -126.5 it is zero (n = -127 leaves no bit); NaN stays NaN.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
    const float kRound = 12582912.f;                 // 1.5 * 2^23: adding it leaves n in the low bits
    const float2 r = __fadd2_rn(x, make_float2(kRound, kRound)), n = __fadd2_rn(r, make_float2(-kRound, -kRound));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 p = __ffma2_rn(make_float2(9.570101276e-3f, 9.570101276e-3f), f, make_float2(5.591785908e-2f, 5.591785908e-2f));
    p = __ffma2_rn(p, f, make_float2(0.2402474433f, 0.2402474433f));
    p = __ffma2_rn(p, f, make_float2(0.6931217909f, 0.6931217909f));
    p = __ffma2_rn(p, f, make_float2(0.9999992847f, 0.9999992847f));
    return __fmul2_rn(p, make_float2(__int_as_float((__float_as_int(r.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(r.y) << 23) + 0x3f800000)));
}
// Two exponentials of the i-th pair of a row: every EVERY-th pair on the FMA pipes, the others on the special function units.
template <int EVERY>
__device__ __forceinline__ float2 exp2_pair(float2 x, int i) {
    return EVERY > 0 && i % (EVERY > 0 ? EVERY : 1) == EVERY - 1 ? exp2_fma(x) : make_float2(ptx::ex2(x.x), ptx::ex2(x.y));
}

// A value that is the same in all lanes, in a form that the compiler knows to be.  The MMA issuer's loops and descriptors then
// live in uniform registers, which the MMA instructions take their operands from: with tiles and rows that come from memory
// (or a warp index from threadIdx) every MMA waited for moves between the register files (dQ kernel at D 128: 855 -> 695 us).
__device__ __forceinline__ int uniform(int x) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)x); }
__device__ __forceinline__ void make_uniform(int& x) { x = uniform(x); }

// One entry of a packed batch's list of work: a tile of a sequence.
struct alignas(32) Item {
    int q0, nq, k0, nk;
    int tile, seq;
    int pad[2];
};
struct alignas(32) ListHead {
    int count;
    int pad[7];
};

// Work of one kernel: tiles of `rows` queries (or keys), the most expensive first, so that the blocks that end last hold short
// ones.  Without a list (batched tensors) tile and sequence follow from the index.
struct WorkList {
    const ListHead* head;             // NULL: no list; items follow the head
    int last;                         // with a list: last_tile of its tiles
    int tiles, S;                     // without a list: tiles per sequence, sequences
    int descending;                   // without a list: whether later tiles are the more expensive ones
};

// The last tile of so many rows that a tensor of the most rows that a call may have (2^30) can hold: its first row fits an int.
constexpr int last_tile(int rows) { return ((1 << 30) - 1) / rows; }
static_assert((int64_t)(last_tile(kTile) + 1) * kTile <= 1 << 30 && (int64_t)(last_tile(2 * kTile) + 1) * 2 * kTile <= 1 << 30, "rows of listed tiles");

__device__ __forceinline__ int list_count(const WorkList& w) { return w.head ? w.head->count : w.tiles * w.S; }

__device__ __forceinline__ void list_item(const CParams& p, const WorkList& w, int i, Seq& s, int& tile) {
    if (w.head) {
        const Item* e = reinterpret_cast<const Item*>(w.head + 1) + i;
        const int4 a = *reinterpret_cast<const int4*>(e);
        // (clipped again: starts that are written to while the list is made may leave entries of it as they were)
        s.b = 0;
        s.q0 = min(max(a.x, 0), p.Nq);
        s.nq = min(max(a.y, 0), p.Nq - s.q0);
        s.k0 = min(max(a.z, 0), p.Nk);
        s.nk = min(max(a.w, 0), p.Nk - s.k0);
        tile = min(max(e->tile, 0), w.last);
        s.id = min(max(e->seq, 0), p.S - 1);
    } else {
        tile = i / w.S;
        s.b = s.id = i - tile * w.S;
        s.q0 = s.k0 = 0;
        s.nq = p.Nq;
        s.nk = p.Nk;
        if (w.descending) tile = w.tiles - 1 - tile;
    }
}

// Key tiles that query tiles of rows [i0, i0 + rows) see; query tiles that see a key of the tile at j0.
__host__ __device__ inline int key_tiles(int i0, int rows, int nq, int nk) {
    if (i0 >= nq) return 0;
    const int last = i0 + rows < nq ? i0 + rows : nq;
    const int seen = last + nk - nq;
    return seen > 0 ? (seen + kTile - 1) / kTile : 0;
}
__host__ __device__ inline int first_query(int j0, int nq, int nk) {       // a multiple of the tile
    const int i = j0 - (nk - nq);
    return i > 0 ? i / kTile * kTile : 0;
}

// The lists of a packed batch, a block for each: tiles of `rows[list]` queries (keys where by_key[list]), sorted by cost in one
// counting pass (4.4 us for 9 sequences of 11 K rows).  Items of equal cost come in any order: it decides where they run, not what they compute.
struct PlanParams {
    ListHead* list[2];
    int rows[2], by_key[2];
    int capacity[2];                  // tiles of sequences that do not overlap (starts that decrease: the rest is left out)
};
constexpr int kPlanBins = 1024;
__global__ void __launch_bounds__(1024) causal_plan_kernel(const CParams p, const PlanParams plan) {
    __shared__ int bins[kPlanBins], warp_sums[32];
    ListHead* const head = plan.list[blockIdx.x];
    const int rows = plan.rows[blockIdx.x], by_key = plan.by_key[blockIdx.x];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    bins[t] = 0;
    __syncthreads();
    auto each = [&](auto&& f) {
        for (int s = warp; s < p.S; s += 32) {
            const Seq q = seq_of(p, s);
            const int n = by_key ? q.nk : q.nq;
            for (int tile = lane; tile * rows < n; tile += 32) {
                const int cost = by_key ? max(ceil_div(q.nq - first_query(tile * rows, q.nq, q.nk), kTile), 0) : key_tiles(tile * rows, rows, q.nq, q.nk);
                f(q, tile, kPlanBins - 1 - min(cost, kPlanBins - 1));
            }
        }
    };
    each([&](const Seq&, int, int bin) { atomicAdd(&bins[bin], 1); });
    __syncthreads();
    // exclusive prefix sum over the bins
    int v = bins[t], x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    x += (warp ? warp_sums[warp - 1] : 0) - v;
    if (t == 1023) head->count = min(max(x + v, 0), plan.capacity[blockIdx.x]);
    bins[t] = x;
    __syncthreads();
    Item* const items = reinterpret_cast<Item*>(head + 1);
    each([&](const Seq& q, int tile, int bin) {
        const int at = atomicAdd(&bins[bin], 1);
        if ((unsigned)at >= (unsigned)plan.capacity[blockIdx.x]) return;
        Item* e = items + at;
        *reinterpret_cast<int4*>(e) = make_int4(q.q0, q.nq, q.k0, q.nk);
        e->tile = tile;
        e->seq = q.id;
    });
}

// Tiles of S sequences that share `rows` rows, at most, and the bytes of a list of so many.
inline int64_t list_capacity(int rows, int tile, int S) { return (int64_t)rows / tile + S; }
inline size_t list_bytes(int64_t items) { return (size_t)(sizeof(ListHead) + items * sizeof(Item) + 255) / 256 * 256; }

}  // namespace causal
}  // namespace sa
