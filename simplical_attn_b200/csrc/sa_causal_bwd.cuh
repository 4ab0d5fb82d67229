// Causal attention backward on the sm_100a tensor cores (bf16 / fp16; head dims as in the forward).
//
//     Delta_i = sum_d dO_id O_id,   P = exp(S - LSE),   dS = scale P (dO V^T - Delta),
//     dV = P^T dO,   dK = dS^T Q,   dQ = dS K.
//
// Two kernels, so that every sum has one owner and a fixed order, without atomics: one owns key tiles and walks over the
// queries that see them, for all query heads of the KV head (dK, dV); one owns query tiles and walks over their keys (dQ).
// That computes S and dO V^T twice: 7 products of 128 x 128 x D per pair of tiles instead of 5.  In exchange nothing is
// written that is not a result, and equal calls give equal bits.
//
// Both are persistent, with groups of four warps (compute) each at a share of a tile's columns and a row of tensor memory per
// thread -- two groups (dK, dV) or four (dQ: 17 % faster at D = 64; for dK, dV no difference) --, then a warp
// issuing MMAs, one TMA loads, one guarding: it zeroes the rows behind a sequence's end in tiles that
// the MMAs sum over (they belong to the next sequence, and a masked zero times its NaN would not be zero) and the queries that see
// no key, and in the dK / dV kernel loads LSE and Delta of the query tile.  P and dS go from registers to tensor memory and from there into the MMA as
// the A operand; a group's packed values lie in the columns of its scores.
//
// The streams of tiles run on over units: while the rows of a finished unit are written out, the next one's scores are
// computed.  MMA cycles per pair of tiles at D = 128: 2048 (dK, dV), 1536 (dQ); exponentials take 1024 of either, and operand reads
// and TMA writes of shared memory 2290 and 1792.
//
// Measured back to back for a second, bf16 B 2 N 8192 H 16/4: D 128 dK, dV 961 us (1144 TFLOP/s of its four products, under the power
// cap; 840 with pauses), dQ 730 us (1130 of three; 670), Delta 42; D 64 660, 492 and 22 us.  In fp16 5 % more at D 128.  Under a
// profiler a step takes about 3220 and 2520 cycles at D 128 (1.64 GHz, tensor pipe 67 and 65 % active), 2590 and 1910 at D 64.
#pragma once

#include "sa_causal_fwd.cuh"

namespace sa {
namespace causal {

constexpr int kColThreads = 384;                     // dK, dV: two compute groups
constexpr int kRowThreads = 640;                     // dQ: four
constexpr int kRowGroups = 4;
constexpr int kRowCols = kTile / kRowGroups;         // columns of a tile that a group of the dQ kernel has
constexpr int kRowWarps = 4 * kRowGroups;            // its compute warps; behind them MMA issuer, TMA, guard
constexpr int kRowRegsCompute = 104, kRowRegsRest = 64;
static_assert(kRowGroups * kRowRegsCompute + kRowRegsRest <= 5 * 96, "register pool of the block (640 x 96 at launch)");
// A operand columns of the k-th step of 16: a group's packed values lie in the first half of its columns.
constexpr int packed_column(int k, int cols) { return k / (cols / 16) * cols + k % (cols / 16) * 8; }
// Every third pair of the dK / dV kernel's exponentials is taken on the FMA pipes: its two groups are in their exponentials at
// the same time (861 -> 841 us at B 2 N 8192 H 16/4 D 128).  In the dQ kernel and the forward that was slower.
constexpr int kFmaCol = 3;

struct BwdParams {
    CParams c;
    WorkList work;            // key tiles (dK, dV) or query tiles (dQ)
    int splits;               // shares of a unit's walk
    const float* lse;
    const float* delta;
    const float2* norms;      // fp16: [sequence][parts] (see ds_factor)
    int parts;
    float* part0;             // splits > 1: [splits][B rows heads][D] partial dQ, or dK
    float* part1;             // dV
    DeviceStatus* status;
    uint64_t wait_limit_ns;
};

// fp16 keeps all of its bits from 2^-14 to 2^16 only.  Over n keys P is about 1 / n and dS that times the size of dO and V, so as they
// are both would lose bits or vanish although the gradients do not (dQ off by 3 % at 4096 keys and |dO| = 10^-3, by 29 % at
// 10^-4).  P therefore goes into dV times 2^12, and dS into dQ and dK without the softmax scale and times a power of two of its
// sequence that brings it to at most 2^12; both are undone in fp32 where rows are written.  (bf16 has the exponents of fp32: nothing
// of this.)  With M the largest |dO_i . V_j| of a sequence, |dS_ij| = P_ij |sum_k P_ik (dP_ij - dP_ik)| <= 2 M P_ij (1 - P_ij) <= M / 2,
// and M is at most the product of the longest rows of dO and V.  For rows of normal values the factor makes dS about 2^10 P.
// 2^12 leaves a factor of 16: scores of 10^7 and more are off by several units in 32 bits, here and in the LSE, and P may be above 1.
// Costs: the longest rows are found by blocks beside Delta's, 2 us at B 2 N 512 H 4 and 8 of 219 for packed sequences of 1999 to 378
// rows (H 16/4 D 64), and 3 % at B 2 N 8192 H 16/4 D 128.
constexpr float kPFactor = 4096.f, kPFactorLog2 = 12.f;
constexpr int kMostParts = 128;
// The factor of a sequence (a whole warp): from the squares of the two lengths a power of two f with sqrt(do2 v2) / 2 f in [2^11, 2^12).
__device__ __forceinline__ float ds_factor(const BwdParams& P, int sequence) {
    float do2 = 0.f, v2 = 0.f;
#pragma unroll
    for (int x = 0; x < kMostParts; x += 32) {         // (loads under way together: this stands at the start of a unit)
        const int y = x + (threadIdx.x & 31);
        const float2 t = y < P.parts ? P.norms[(int64_t)sequence * P.parts + y] : make_float2(0.f, 0.f);
        do2 = fmaxf(do2, t.x);
        v2 = fmaxf(v2, t.y);
    }
    // (not negative: ordered as their bits are)
    do2 = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(do2)));
    v2 = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v2)));
    const float x = do2 * v2;                          // (2^-96 to 2^79)
    if (!(x > 0.f)) return 1.f;
    const int e = (__float_as_int(x) >> 23) - 127;     // x < 2^(e + 1)
    return __int_as_float((13 - ((e + 2) >> 1) + 127) << 23);
}

__device__ __forceinline__ float one_over(float power_of_two) { return __int_as_float((254 << 23) - __float_as_int(power_of_two)); }

// Squares of the longest rows of dO and V of every sequence, without elements that are not finite (their rows' gradients are not
// either) and queries that see nothing: `parts` blocks for a sequence.
template <int HD>
__device__ __forceinline__ void longest_rows(const CParams& p, const __nv_bfloat16* __restrict__ v, const __nv_bfloat16* __restrict__ d_o,
                                             float2* __restrict__ norms, int parts) {
    using E = ptx::El<true>;
    constexpr int kLanes = HD / 8, kRows = 256 / kLanes, kUnroll = 4;
    __shared__ float tops[2][8];
    const int lane = threadIdx.x % kLanes, row0 = threadIdx.x / kLanes;
    const Seq s = seq_of(p, blockIdx.x / parts);
    const unsigned part = blockIdx.x % parts;
    auto longest = [&](const __nv_bfloat16* x, const sa_strides& st, int first, int rows, unsigned heads) {
        const unsigned total = (unsigned)max(rows - first, 0) * heads;         // (rows fit 31 bits)
        float top = 0.f;
        x += s.b * st.b + 8 * lane;
        for (unsigned r0 = part * kRows * kUnroll; r0 < total; r0 += parts * kRows * kUnroll) {
            uint4 w[kUnroll];
#pragma unroll
            for (int y = 0; y < kUnroll; ++y) {
                const unsigned r = r0 + y * kRows + row0, i = r / heads;
                w[y] = make_uint4(0, 0, 0, 0);
                if (r < total && 8 * lane < p.D) w[y] = *reinterpret_cast<const uint4*>(x + (int64_t)(first + (int)i) * st.n + (r - i * heads) * st.h);
            }
#pragma unroll
            for (int y = 0; y < kUnroll; ++y) {
                const uint32_t word[4] = {w[y].x, w[y].y, w[y].z, w[y].w};
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = E::lo(word[e]), b = E::hi(word[e]);
                    if (fabsf(a) < INFINITY) sum = fmaf(a, a, sum);
                    if (fabsf(b) < INFINITY) sum = fmaf(b, b, sum);
                }
#pragma unroll
                for (int z = kLanes / 2; z > 0; z >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, z);
                top = fmaxf(top, sum);
            }
        }
#pragma unroll
        for (int z = 16; z > 0; z >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
        return top;
    };
    const float a = longest(d_o + s.q0 * p.d_o.n, p.d_o, max(-s.off(), 0), s.nq, p.H), b = longest(v + s.k0 * p.v.n, p.v, 0, s.nk, p.Hkv);
    if ((threadIdx.x & 31) == 0) {
        tops[0][threadIdx.x >> 5] = a;
        tops[1][threadIdx.x >> 5] = b;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float2 t = make_float2(0.f, 0.f);
        for (int y = 0; y < 8; ++y) t = make_float2(fmaxf(t.x, tops[0][y]), fmaxf(t.y, tops[1][y]));
        norms[blockIdx.x] = t;
    }
}

// Delta, eight elements a lane; for fp16 the first blocks find the sequences' longest rows.
template <int HD, bool F16>
__global__ void __launch_bounds__(256) causal_delta16_kernel(const CParams p, const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ o_low,
                                                            const __nv_bfloat16* __restrict__ v, const __nv_bfloat16* __restrict__ d_o, float* __restrict__ delta,
                                                            float2* __restrict__ norms, int parts) {
    using E = ptx::El<F16>;
    constexpr int kLanes = HD / 8;
    const int lane = threadIdx.x % kLanes;
    // (rows fit 31 bits; 64-bit divisions took most of this kernel's time)
    unsigned block = blockIdx.x;
    if constexpr (F16) {
        const unsigned first = (unsigned)p.S * (unsigned)parts;
        if (block < first) {
            longest_rows<HD>(p, v, d_o, norms, parts);
            return;
        }
        block -= first;
    }
    const unsigned w = block * (256 / kLanes) + threadIdx.x / kLanes;
    float sum = 0.f;
    int h = 0, i = 0, b = 0;
    const bool in = w < (unsigned)(p.B * p.Nq * p.H);
    if (in) {
        const unsigned bi = w / (unsigned)p.H;
        h = (int)(w - bi * (unsigned)p.H);
        b = (int)(bi / (unsigned)p.Nq);
        i = (int)(bi - (unsigned)b * (unsigned)p.Nq);
        const int64_t at = b * p.o.b + i * p.o.n + h * p.o.h + 8 * lane;
        const uint4 none = make_uint4(0, 0, 0, 0);
        const bool col = 8 * lane < p.D;
        const uint4 x = col ? *reinterpret_cast<const uint4*>(o + at) : none, z = col && o_low ? *reinterpret_cast<const uint4*>(o_low + at) : none;
        const uint4 y = col ? *reinterpret_cast<const uint4*>(d_o + b * p.d_o.b + i * p.d_o.n + h * p.d_o.h + 8 * lane) : none;
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum = fmaf(E::lo(xw[e]) + E::lo(zw[e]), E::lo(yw[e]), sum);
            sum = fmaf(E::hi(xw[e]) + E::hi(zw[e]), E::hi(yw[e]), sum);
        }
    }
#pragma unroll
    for (int s = kLanes / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (in && lane == 0) delta[((int64_t)b * p.H + h) * p.Nq + i] = sum;
}

// Units in the order of the work list, a block's rounds in alternating direction.
struct Walk {
    int u, round, count;
    __device__ __forceinline__ Walk(const BwdParams& P, int heads) {
        count = list_count(P.work) * heads * P.splits;
        round = 0;
        u = blockIdx.x;
    }
    __device__ __forceinline__ bool valid() const { return u < count; }
    __device__ __forceinline__ void next() {
        ++round;
        u = round * (int)gridDim.x + ((round & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
    }
};

#define SA_ARRIVE(OFF, BASE)                       \
    do {                                           \
        __syncwarp();                              \
        if (lane == 0) mbar_arrive<(OFF)>(BASE);   \
    } while (0)

// Zeroes the rows of a [128 x HD] tile that are not in [first, from) (a warp).
template <int HD>
__device__ __forceinline__ void zero_tile_rows(uint32_t tile, int first, int from, int lane) {
    for (int c = lane; c < kTile * HD / 8; c += 32)
        if (c / 8 % kTile < first || c / 8 % kTile >= from) ptx::sts128(tile + c * 16, make_uint4(0, 0, 0, 0));
}

// ---------------------------------------------------------------------------------------------- dK, dV
template <int HD>
struct ColLayout {
    static constexpr int kSlabs = HD / 64;
    static constexpr int kSlab = kTile * 128;
    static constexpr int kTileBytes = kSlabs * kSlab;
    static constexpr int kStages = HD == 128 ? 2 : 4;        // Q and dO tiles in flight
    static constexpr int kMisc = 256;
    static constexpr int kStats = 512;                       // [stage][LSE, Delta][128] floats
    static constexpr int kK = 512 + 4 * 2 * kTile * 4 + 512; // 5120
    static constexpr int kV = kK + kTileBytes;
    static constexpr int kRing = kV + kTileBytes;
    static constexpr int kBytes = kRing + kStages * 2 * kTileBytes + 1024;
    static_assert(kK % 1024 == 0 && kStats + kStages * 2 * kTile * 4 <= kK && kBytes <= 227 * 1024, "shared memory of a block");
};

// A unit: key tile at j0 of a KV head, steps it0 .. it0 + n of (query head of the group, query tile).
struct ColUnit {
    Seq s;
    int hk, split, j0, first, tiles, it0, n;
};
__device__ __forceinline__ ColUnit col_unit(const BwdParams& P, const Walk& w) {
    ColUnit r;
    const int x = w.u / P.splits, item = x / P.c.Hkv;
    r.split = w.u - x * P.splits;
    r.hk = x - item * P.c.Hkv;
    int tile;
    list_item(P.c, P.work, item, r.s, tile);
    r.j0 = tile * kTile;
    r.first = first_query(r.j0, r.s.nq, r.s.nk);
    r.tiles = r.s.nq > r.first && r.j0 < r.s.nk ? (r.s.nq - r.first + kTile - 1) / kTile : 0;
    const int total = r.tiles * P.c.G, share = (total + P.splits - 1) / P.splits;
    r.it0 = r.split * share;
    r.n = min(max(total - r.it0, 0), share);
    return r;
}
// Position in a unit's walk.
struct ColStep {
    int g, qt;               // query head of the group, query tile
    __device__ __forceinline__ explicit ColStep(const ColUnit& u) : g(u.tiles ? u.it0 / u.tiles : 0), qt(u.it0 - g * u.tiles) {}
    __device__ __forceinline__ void next(const ColUnit& u) {
        if (++qt == u.tiles) {
            qt = 0;
            ++g;
        }
    }
    __device__ __forceinline__ int i0(const ColUnit& u) const { return u.first + qt * kTile; }
};

template <int HD, bool F16>
__global__ void __launch_bounds__(kColThreads, 1)
causal_dkv_tc_kernel(const __grid_constant__ BwdParams P, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, __nv_bfloat16* __restrict__ dk,
                     __nv_bfloat16* __restrict__ dv) {
    using L = ColLayout<HD>;
    using namespace ptx;
    using E = El<F16>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem);
    const CParams& p = P.c;

    constexpr int kFull = 0;                          // [stage] Q and dO landed
    constexpr int kEmpty = kFull + 8 * L::kStages;    //         read by the unit's MMAs
    constexpr int kPassed = kEmpty + 8 * L::kStages;  //         guarded, LSE and Delta there
    constexpr int kKvFull = kPassed + 8 * L::kStages; // K and V of the unit landed
    constexpr int kKvFree = kKvFull + 8;              //         ... read by its last S and dP MMAs
    constexpr int kSReady = kKvFree + 8;
    constexpr int kPReady = kSReady + 8;
    constexpr int kDpReady = kPReady + 8;
    constexpr int kDsReady = kDpReady + 8;
    constexpr int kAccReady = kDsReady + 8;           // dK and dV final
    constexpr int kAccFree = kAccReady + 8;           //         ... read out
    static_assert(kAccFree + 8 <= L::kMisc, "room for the barriers");
    uint32_t* tmem_slot = (uint32_t*)(smem + L::kMisc);
    const WaitCtx wctx{base + L::kMisc + 4, P.status, P.wait_limit_ns};

    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    if (tid == 0) {
        auto init = [&](int off, int n, uint32_t count) {
            for (int x = 0; x < n; ++x) mbar_init((uint64_t*)(smem + off) + x, count);
        };
        init(kFull, 3 * L::kStages, 1);
        init(kKvFull, 2, 1);
        init(kSReady, 1, 1);
        init(kPReady, 1, 8);
        init(kDpReady, 1, 1);
        init(kDsReady, 1, 8);
        init(kAccReady, 1, 1);
        init(kAccFree, 1, 8);
        *(volatile int*)(smem + L::kMisc + 4) = 0;
        fence_mbar_init();
    }
    if (warp == 8) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);
    const uint32_t tm_s = tmem, tm_dp = tmem + kTile, tm_dv = tmem + 2 * kTile, tm_dk = tm_dv + HD;

    if (warp >= 8) {
        reg_dealloc<kFwdRegsRest>();
        if (warp == 9) {
            // ---------------------------------------------------------------- TMA
            if (lane == 0) {
                prefetch_tensormap(&map_q);
                prefetch_tensormap(&map_k);
                prefetch_tensormap(&map_v);
                prefetch_tensormap(&map_do);
                Ring g;
                uint32_t nu = 0;
                for (Walk w(P, p.Hkv); w.valid(); w.next()) {
                    const ColUnit u = col_unit(P, w);
                    if (u.n == 0) continue;
                    auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head) {
#pragma unroll
                        for (int sl = 0; sl < L::kSlabs; ++sl) tma_load_4d(dst + sl * L::kSlab, map, bar, sl * 64, row, head, u.s.b);
                    };
                    ColStep st(u);
                    for (int it = 0; it < u.n; ++it, st.next(u)) {
                        mbar_wait<kEmpty>(base + 8 * g.s, g.phase ^ 1, wctx, 2);
                        const uint32_t bar = base + kFull + 8 * g.s, dst = base + L::kRing + g.s * 2 * L::kTileBytes;
                        mbar_arrive_expect_tx(bar, 2 * L::kTileBytes);
                        const int row = u.s.q0 + st.i0(u), h = u.hk * p.G + st.g;
                        load(dst, &map_q, bar, row, h);
                        load(dst + L::kTileBytes, &map_do, bar, row, h);
                        g.next<L::kStages>();
                        if (it == 0) {
                            mbar_wait<kKvFree>(base, (nu & 1) ^ 1, wctx, 1);
                            mbar_arrive_expect_tx(base + kKvFull, 2 * L::kTileBytes);
                            load(base + L::kK, &map_k, base + kKvFull, u.s.k0 + u.j0, u.hk);
                            load(base + L::kV, &map_v, base + kKvFull, u.s.k0 + u.j0, u.hk);
                            ++nu;
                        }
                    }
                }
            }
            __syncwarp();
        } else if (warp == 8) {
            // ---------------------------------------------------------------- MMA issuer:  dV(n), S(n + 1), dK(n), dP(n + 1)
            const uint32_t leader = elect_one();
            const uint32_t idesc_s = make_idesc(128, kTile, false, false, F16), idesc_d = make_idesc(128, HD, false, true, F16);
            auto scores = [&](uint32_t d, uint32_t a_tile, uint32_t b_tile) {        // d = A . B^T, both K-major
                const uint32_t da = desc_lo(a_tile, 16), db = desc_lo(b_tile, 16);
                static_for<HD / 16>([&](auto kk_c) {
                    constexpr int kk = decltype(kk_c)::value, off = ((kk >> 2) * L::kSlab + (kk & 3) * 32) >> 4;
                    mma_ss_lo<off, off>(leader, d, da, db, idesc_s, kk > 0);
                });
            };
            auto sums = [&](uint32_t d, uint32_t a, uint32_t b_tile, bool first) {   // d += A . B, A packed in tensor memory
                const uint32_t db = desc_lo(b_tile, L::kSlab);
                static_for<8>([&](auto kk_c) {
                    constexpr int kk = decltype(kk_c)::value;
                    mma_ts_lo<packed_column(kk, kTile / 2), kk * (2048 >> 4)>(leader, d, a, db, idesc_d, !first || kk > 0);
                });
            };
            auto stage = [&](const Ring& g) { return base + L::kRing + g.s * 2 * L::kTileBytes; };
            auto issue_s = [&](const Ring& g) {
                mbar_wait<kFull>(base + 8 * g.s, g.phase, wctx, 4);
                mbar_wait<kPassed>(base + 8 * g.s, g.phase, wctx, 5);
                tc_fence_after();
                scores(tm_s, base + L::kK, stage(g));
                tc_commit<kSReady>(leader, base);
            };
            auto issue_dp = [&](const Ring& g, bool last) {
                scores(tm_dp, base + L::kV, stage(g) + L::kTileBytes);
                tc_commit<kDpReady>(leader, base);
                if (last) tc_commit<kKvFree>(leader, base);
            };
            Ring g;
            uint32_t n = 0, nu = 0;
            Walk w(P, p.Hkv);
            make_uniform(w.count);
            for (; w.valid(); w.next()) {
                ColUnit u = col_unit(P, w);
                make_uniform(u.n);
                if (u.n == 0) continue;
                mbar_wait<kKvFull>(base, nu & 1, wctx, 3);
                issue_s(g);
                issue_dp(g, u.n == 1);
#pragma unroll 1
                for (int it = 0; it < u.n; ++it, ++n) {
                    Ring gn = g;
                    gn.next<L::kStages>();
                    if (it == 0 && nu > 0) mbar_wait<kAccFree>(base, (nu - 1) & 1, wctx, 6);
                    mbar_wait<kPReady>(base, n & 1, wctx, 7);
                    tc_fence_after();
                    sums(tm_dv, tm_s, stage(g) + L::kTileBytes, it == 0);
                    if (it + 1 < u.n) issue_s(gn);
                    mbar_wait<kDsReady>(base, n & 1, wctx, 8);
                    tc_fence_after();
                    sums(tm_dk, tm_dp, stage(g), it == 0);
                    tc_commit<kEmpty>(leader, base + 8 * g.s);
                    if (it + 1 < u.n) issue_dp(gn, it + 2 == u.n);
                    else tc_commit<kAccReady>(leader, base);
                    g = gn;
                }
                ++nu;
            }
        } else if (warp == 10) {
            // ---------------------------------------------------------------- guard; LSE and Delta
            Ring g;
            for (Walk w(P, p.Hkv); w.valid(); w.next()) {
                const ColUnit u = col_unit(P, w);
                ColStep st(u);
                const float f = F16 ? ds_factor(P, u.s.id) / kPFactor : p.scale;
                for (int it = 0; it < u.n; ++it, st.next(u)) {
                    const int i0 = st.i0(u), h = u.hk * p.G + st.g;
                    const int64_t at = ((int64_t)u.s.b * p.H + h) * p.Nq + u.s.q0 + i0;
                    float ls[4], dl[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 32 * e + lane;
                        const bool in = i0 + i < u.s.nq && i0 + i + u.s.off() >= 0;
                        ls[e] = in ? P.lse[at + i] : -INFINITY;
                        dl[e] = in ? P.delta[at + i] : 0.f;
                    }
                    mbar_wait<kFull>(base + 8 * g.s, g.phase, wctx, 9);
                    // (a row that does not exist, sees nothing or has scores of -inf only has P = exp2(-inf) = 0)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        dl[e] = ls[e] == -INFINITY ? 0.f : dl[e] * f;
                        ls[e] = ls[e] == -INFINITY ? INFINITY : ls[e] * kLog2e - (F16 ? kPFactorLog2 : 0.f);
                    }
                    const uint32_t stats = base + L::kStats + g.s * 2 * kTile * 4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sts_f32(stats + (32 * e + lane) * 4, ls[e]);
                        sts_f32(stats + (kTile + 32 * e + lane) * 4, dl[e]);
                    }
                    const int blind = -(i0 + u.s.off());        // rows before it see no key (there are some if queries outnumber keys)
                    if (i0 + kTile > u.s.nq || blind > 0) {
                        const uint32_t tile = base + L::kRing + g.s * 2 * L::kTileBytes;
                        zero_tile_rows<HD>(tile, blind, u.s.nq - i0, lane);
                        zero_tile_rows<HD>(tile + L::kTileBytes, blind, u.s.nq - i0, lane);
                        fence_proxy_async_smem();
                    }
                    SA_ARRIVE(kPassed, base + 8 * g.s);
                    g.next<L::kStages>();
                }
            }
        }
    } else {
        // -------------------------------------------------------------------- compute: a key per thread, 64 queries per group
        reg_alloc<kFwdRegsSoftmax>();
        const int grp = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(row & ~31) << 16;
        const uint32_t s_addr = tm_s + lanes + 64 * grp, dp_addr = tm_dp + lanes + 64 * grp;
        const float2 c2 = make_float2(p.scale * kLog2e, p.scale * kLog2e);
        Ring g;
        uint32_t n = 0, nu = 0;
        for (Walk w(P, p.Hkv); w.valid(); w.next()) {
            const ColUnit u = col_unit(P, w);
            ColStep st(u);
            const float f = F16 ? ds_factor(P, u.s.id) / kPFactor : p.scale;        // of dP; P has its factor already (through its LSE)
            const float2 sc = make_float2(f, f);
#pragma unroll 1
            for (int it = 0; it < u.n; ++it, ++n, st.next(u)) {
                const int i0 = st.i0(u);
                const uint32_t stats = base + L::kStats + g.s * 2 * kTile * 4 + grp * 64 * 4;
                mbar_wait<kPassed>(base + 8 * g.s, g.phase, wctx, 10);
                mbar_wait<kSReady>(base, n & 1, wctx, 11);
                tc_fence_after();
                float pr[64];
                auto load = [&](uint32_t addr) {
                    tmem_ld32(addr, reinterpret_cast<uint32_t(&)[32]>(pr[0]));
                    tmem_ld32(addr + 32, reinterpret_cast<uint32_t(&)[32]>(pr[32]));
                    tmem_wait_ld();
                };
                load(s_addr);
                // query i sees key j if j <= i + off: columns from `lo` on
                const int lo = u.j0 + row - u.s.off() - i0 - 64 * grp;
                const bool masked = u.j0 + kTile - 1 > i0 + u.s.off();
                uint32_t seen[2] = {~0u, ~0u};
                if (masked) {
                    seen[0] = lo <= 0 ? ~0u : lo >= 32 ? 0u : ~0u << lo;
                    seen[1] = lo <= 32 ? ~0u : lo >= 64 ? 0u : ~0u << (lo - 32);
                }
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const uint4 x = lds128(stats + c * 4);
                    const float2 y0 = __ffma2_rn(make_float2(pr[c], pr[c + 1]), c2, make_float2(-__uint_as_float(x.x), -__uint_as_float(x.y)));
                    const float2 y1 = __ffma2_rn(make_float2(pr[c + 2], pr[c + 3]), c2, make_float2(-__uint_as_float(x.z), -__uint_as_float(x.w)));
                    const float2 e0 = exp2_pair<kFmaCol>(y0, c / 2), e1 = exp2_pair<kFmaCol>(y1, c / 2 + 1);
                    pr[c] = e0.x;
                    pr[c + 1] = e0.y;
                    pr[c + 2] = e1.x;
                    pr[c + 3] = e1.y;
                }
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) pr[c] = (seen[c >> 5] >> (c & 31)) & 1 ? pr[c] : 0.f;
                }
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) pk[e] = E::pack(pr[c + 2 * e], pr[c + 2 * e + 1]);
                    tmem_st16(s_addr + c / 2, pk);
                }
                tmem_wait_st();
                tc_fence_before();
                SA_ARRIVE(kPReady, base);
                mbar_wait<kDpReady>(base, n & 1, wctx, 12);
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    uint32_t v[32], pk[16];
                    tmem_ld32(dp_addr + c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const uint4 x = lds128(stats + (kTile + c + e) * 4);
                        float2 y0 = __ffma2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc, make_float2(-__uint_as_float(x.x), -__uint_as_float(x.y)));
                        float2 y1 = __ffma2_rn(make_float2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), sc, make_float2(-__uint_as_float(x.z), -__uint_as_float(x.w)));
                        y0 = __fmul2_rn(y0, make_float2(pr[c + e], pr[c + e + 1]));
                        y1 = __fmul2_rn(y1, make_float2(pr[c + e + 2], pr[c + e + 3]));
                        if (masked) {
                            const uint32_t bits = seen[c >> 5] >> e;
                            y0.x = bits & 1 ? y0.x : 0.f;
                            y0.y = bits & 2 ? y0.y : 0.f;
                            y1.x = bits & 4 ? y1.x : 0.f;
                            y1.y = bits & 8 ? y1.y : 0.f;
                        }
                        pk[e >> 1] = E::pack(y0.x, y0.y);
                        pk[(e >> 1) + 1] = E::pack(y1.x, y1.y);
                    }
                    // (the 16 packed columns lie in those of the first 32 products, which are in registers by now)
                    tmem_st16(dp_addr + c / 2, pk);
                }
                tmem_wait_st();
                tc_fence_before();
                SA_ARRIVE(kDsReady, base);
                g.next<L::kStages>();
            }
            // ---- group 0 writes dV, group 1 dK
            __nv_bfloat16* const out = grp ? dk : dv;
            const sa_strides so = grp ? p.dk : p.dv;
            float* const part = grp ? P.part0 : P.part1;
            const bool mine = u.j0 + row < u.s.nk && out != nullptr;
            const uint32_t a_addr = (grp ? tm_dk : tm_dv) + lanes;
            if (u.n > 0) {
                mbar_wait<kAccReady>(base, nu & 1, wctx, 13);
                tc_fence_after();
                ++nu;
            }
            const float undo = grp ? p.scale * one_over(f * kPFactor) : 1.f / kPFactor;
            __nv_bfloat16* const dst = out + u.s.b * so.b + (int64_t)(u.s.k0 + u.j0 + row) * so.n + u.hk * so.h;
            float* const pdst = part + (((int64_t)u.split * p.B + u.s.b) * p.Hkv + u.hk) * (int64_t)p.Nk * HD + (int64_t)(u.s.k0 + u.j0 + row) * HD;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t x[32];
                if (u.n > 0) {
                    tmem_ld32(a_addr + c0, x);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = 0u;
                }
                if (!mine) continue;
                if constexpr (F16) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * undo);
                }
                if (P.splits > 1) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(pdst + c0 + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        if (c0 + e < p.D)
                            *reinterpret_cast<uint4*>(dst + c0 + e) =
                                make_uint4(E::pack(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), E::pack(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])),
                                           E::pack(__uint_as_float(x[e + 4]), __uint_as_float(x[e + 5])), E::pack(__uint_as_float(x[e + 6]), __uint_as_float(x[e + 7])));
                }
            }
            if (u.n > 0) {
                tc_fence_before();
                SA_ARRIVE(kAccFree, base);
            }
        }
    }
    if (p.cu_k != nullptr && P.splits == 1) {
        if (dk) zero_outside(dk, p.dk, p.Hkv, p.D, p.Nk, p.cu_k, p.S, blockIdx.x, gridDim.x);
        if (dv) zero_outside(dv, p.dv, p.Hkv, p.D, p.Nk, p.cu_k, p.S, blockIdx.x, gridDim.x);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------------------------- dQ
template <int HD>
struct RowLayout {
    static constexpr int kSlabs = HD / 64;
    static constexpr int kSlab = kTile * 128;
    static constexpr int kTileBytes = kSlabs * kSlab;
    static constexpr int kKStages = HD == 128 ? 3 : 5;
    static constexpr int kVStages = HD == 128 ? 2 : 4;
    static constexpr int kMisc = 384;
    static constexpr int kQ = 2048;
    static constexpr int kDo = kQ + kTileBytes;
    static constexpr int kKRing = kDo + kTileBytes;
    static constexpr int kVRing = kKRing + kKStages * kTileBytes;
    static constexpr int kBytes = kVRing + kVStages * kTileBytes + 1024;
    static_assert(kQ % 1024 == 0 && kBytes <= 227 * 1024, "shared memory of a block");
};

// A unit: query tile at i0 of a head, key tiles t0 .. t0 + n.
struct RowUnit {
    Seq s;
    int h, split, i0, t0, n;
    __device__ __forceinline__ int first_masked() const {         // counted from t0
        const int limit = i0 + s.off() + 1;
        return max((limit > 0 ? limit : 0) / kTile - t0, 0);
    }
};
__device__ __forceinline__ RowUnit row_unit(const BwdParams& P, const Walk& w) {
    RowUnit r;
    const int x = w.u / P.splits, item = x / P.c.H;
    r.split = w.u - x * P.splits;
    r.h = x - item * P.c.H;
    int tile;
    list_item(P.c, P.work, item, r.s, tile);
    r.i0 = tile * kTile;
    const int total = key_tiles(r.i0, kTile, r.s.nq, r.s.nk), share = (total + P.splits - 1) / P.splits;
    r.t0 = r.split * share;
    r.n = min(max(total - r.t0, 0), share);
    return r;
}
// The stream of tiles of all units of a block.
struct RowStream {
    Walk w;
    RowUnit u;
    int t;
    __device__ __forceinline__ explicit RowStream(const BwdParams& P) : w(P, P.c.H), t(0) { settle(P); }
    __device__ __forceinline__ void settle(const BwdParams& P) {          // at w's unit, or the next that has tiles
        while (w.valid()) {
            u = row_unit(P, w);
            if (u.n > 0) return;
            w.next();
        }
    }
    __device__ __forceinline__ bool valid() const { return w.valid(); }
    __device__ __forceinline__ void next(const BwdParams& P) {
        if (++t == u.n) {
            t = 0;
            w.next();
            settle(P);
        }
    }
};

template <int HD, bool F16>
__global__ void __launch_bounds__(kRowThreads, 1)
causal_dq_tc_kernel(const __grid_constant__ BwdParams P, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, __nv_bfloat16* __restrict__ dq) {
    using L = RowLayout<HD>;
    using namespace ptx;
    using E = El<F16>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem);
    const CParams& p = P.c;

    constexpr int kKFull = 0;                           // [stage]
    constexpr int kKEmpty = kKFull + 8 * L::kKStages;
    constexpr int kPassed = kKEmpty + 8 * L::kKStages;
    constexpr int kVFull = kPassed + 8 * L::kKStages;
    constexpr int kVEmpty = kVFull + 8 * L::kVStages;
    constexpr int kQFull = kVEmpty + 8 * L::kVStages;
    constexpr int kQFree = kQFull + 8;                  // the unit's last S has read Q
    constexpr int kDoFull = kQFree + 8;
    constexpr int kDoFree = kDoFull + 8;                // its last dP has read dO
    // [2], by parity of the tile: MMAs and compute run up to two tiles apart
    constexpr int kSReady = kDoFree + 8;
    constexpr int kSRead = kSReady + 16;                // S is in registers: its columns may take dP
    constexpr int kDpReady = kSRead + 16;
    constexpr int kDsReady = kDpReady + 16;
    constexpr int kAccReady = kDsReady + 16;
    constexpr int kAccFree = kAccReady + 8;
    static_assert(kAccFree + 8 <= L::kMisc, "room for the barriers");
    uint32_t* tmem_slot = (uint32_t*)(smem + L::kMisc);
    const WaitCtx wctx{base + L::kMisc + 4, P.status, P.wait_limit_ns};

    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    if (tid == 0) {
        auto init = [&](int off, int n, uint32_t count) {
            for (int x = 0; x < n; ++x) mbar_init((uint64_t*)(smem + off) + x, count);
        };
        init(kKFull, L::kKStages, 1);
        init(kKEmpty, L::kKStages, 2);
        init(kPassed, L::kKStages, 1);
        init(kVFull, 2 * L::kVStages, 1);
        init(kQFull, 4, 1);
        init(kSReady, 2, 1);
        init(kSRead, 2, kRowWarps);
        init(kDpReady, 2, 1);
        init(kDsReady, 2, kRowWarps);
        init(kAccReady, 1, 1);
        init(kAccFree, 1, kRowWarps);
        *(volatile int*)(smem + L::kMisc + 4) = 0;
        fence_mbar_init();
    }
    if (warp == kRowWarps) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);
    // Three slots of 128 columns: S of tile n in slot -n mod 3, dP of tile n where S of tile n - 1 was (slot 1 - n mod 3), S of
    // the next tile in the third.
    const uint32_t tm_dq = tmem + 3 * kTile;
    auto s_slot = [](uint32_t m3) { return m3 == 0 ? 0u : 3u - m3; };
    auto dp_slot = [](uint32_t m3) { return m3 == 0 ? 1u : m3 == 1 ? 0u : 2u; };

    if (warp >= kRowWarps) {
        reg_dealloc<kRowRegsRest>();
        if (warp == kRowWarps + 1) {
            // ---------------------------------------------------------------- TMA
            if (lane == 0) {
                prefetch_tensormap(&map_q);
                prefetch_tensormap(&map_k);
                prefetch_tensormap(&map_v);
                prefetch_tensormap(&map_do);
                Ring gk, gv;
                uint32_t nu = 0;
                for (RowStream x(P); x.valid(); x.next(P)) {
                    const RowUnit& u = x.u;
                    auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head) {
                        mbar_arrive_expect_tx(bar, L::kTileBytes);
#pragma unroll
                        for (int sl = 0; sl < L::kSlabs; ++sl) tma_load_4d(dst + sl * L::kSlab, map, bar, sl * 64, row, head, u.s.b);
                    };
                    const int row = u.s.k0 + (u.t0 + x.t) * kTile, hk = u.h / p.G;
                    mbar_wait<kKEmpty>(base + 8 * gk.s, gk.phase ^ 1, wctx, 1);
                    load(base + L::kKRing + gk.s * L::kTileBytes, &map_k, base + kKFull + 8 * gk.s, row, hk);
                    gk.next<L::kKStages>();
                    if (x.t == 0) {
                        mbar_wait<kQFree>(base, (nu & 1) ^ 1, wctx, 2);
                        load(base + L::kQ, &map_q, base + kQFull, u.s.q0 + u.i0, u.h);
                    }
                    mbar_wait<kVEmpty>(base + 8 * gv.s, gv.phase ^ 1, wctx, 3);
                    load(base + L::kVRing + gv.s * L::kTileBytes, &map_v, base + kVFull + 8 * gv.s, row, hk);
                    gv.next<L::kVStages>();
                    if (x.t == 0) {
                        mbar_wait<kDoFree>(base, (nu & 1) ^ 1, wctx, 4);
                        load(base + L::kDo, &map_do, base + kDoFull, u.s.q0 + u.i0, u.h);
                        ++nu;
                    }
                }
            }
            __syncwarp();
        } else if (warp == kRowWarps) {
            // ---------------------------------------------------------------- MMA issuer:  dP(n + 1), dQ(n), S(n + 2)
            const uint32_t leader = elect_one();
            const uint32_t idesc_s = make_idesc(128, kTile, false, false, F16), idesc_d = make_idesc(128, HD, false, true, F16);
            auto scores = [&](uint32_t d, uint32_t a_tile, uint32_t b_tile) {
                const uint32_t da = desc_lo(a_tile, 16), db = desc_lo(b_tile, 16);
                static_for<HD / 16>([&](auto kk_c) {
                    constexpr int kk = decltype(kk_c)::value, off = ((kk >> 2) * L::kSlab + (kk & 3) * 32) >> 4;
                    mma_ss_lo<off, off>(leader, d, da, db, idesc_s, kk > 0);
                });
            };
            // Three positions in the one stream of tiles: S is up to two tiles ahead of dQ, dP one.  S finds the units and leaves
            // their numbers of tiles (0: no more) for the others, by unit modulo 4.
            Walk w(P, p.H);
            make_uniform(w.count);
            int n0 = 0, n1 = 0, n2 = 0, n3 = 0;
            auto tiles_of = [&](uint32_t u) { return u & 2 ? (u & 1 ? n3 : n2) : (u & 1 ? n1 : n0); };
            uint32_t us = 0, up = 0, uq = 0;                             // units
            int ts = 0, tp = 0, tq = 0;                                  // tiles of theirs
            Ring gs, gp, gq;
            uint32_t ns = 0, np = 0, n = 0, s3 = 0, p3 = 0, q3 = 0;      // tiles so far, also modulo 3
            auto find = [&] {
                int x = 0;
                for (; w.valid() && x == 0; w.next()) x = uniform(row_unit(P, w).n);
                if ((us & 3) == 0) n0 = x;
                else if ((us & 3) == 1) n1 = x;
                else if ((us & 3) == 2) n2 = x;
                else n3 = x;
            };
            auto issue_s = [&] {
                const int tiles = tiles_of(us);
                if (tiles == 0) return;
                const bool last = ts == tiles - 1;
                if (ts == 0) mbar_wait<kQFull>(base, us & 1, wctx, 5);
                mbar_wait<kKFull>(base + 8 * gs.s, gs.phase, wctx, 6);
                if (last) mbar_wait<kPassed>(base + 8 * gs.s, gs.phase, wctx, 7);      // (keys may end within the last tile)
                tc_fence_after();
                scores(tmem + s_slot(s3) * kTile, base + L::kQ, base + L::kKRing + gs.s * L::kTileBytes);
                if (ns & 1) tc_commit<kSReady + 8>(leader, base);
                else tc_commit<kSReady>(leader, base);
                gs.next<L::kKStages>();
                ++ns;
                s3 = s3 == 2 ? 0 : s3 + 1;
                ++ts;
                if (last) {
                    tc_commit<kQFree>(leader, base);
                    ts = 0;
                    ++us;
                    find();
                }
            };
            auto issue_dp = [&] {
                const int tiles = tiles_of(up);
                if (tiles == 0) return;
                if (tp == 0) mbar_wait<kDoFull>(base, up & 1, wctx, 8);
                mbar_wait<kVFull>(base + 8 * gp.s, gp.phase, wctx, 9);
                if (np > 0) mbar_wait<kSRead>(base + 8 * ((np - 1) & 1), ((np - 1) >> 1) & 1, wctx, 10);     // S of the tile before is in registers
                tc_fence_after();
                scores(tmem + dp_slot(p3) * kTile, base + L::kDo, base + L::kVRing + gp.s * L::kTileBytes);
                if (np & 1) tc_commit<kDpReady + 8>(leader, base);
                else tc_commit<kDpReady>(leader, base);
                tc_commit<kVEmpty>(leader, base + 8 * gp.s);
                gp.next<L::kVStages>();
                ++np;
                p3 = p3 == 2 ? 0 : p3 + 1;
                if (++tp == tiles) {
                    tc_commit<kDoFree>(leader, base);
                    tp = 0;
                    ++up;
                }
            };
            find();
            issue_s();
            issue_dp();
            issue_s();
#pragma unroll 1
            for (int tiles = tiles_of(0); tiles > 0;) {
                // (at the end of a unit dQ goes first: dP of the next unit still waits for its dO)
                const bool last = tq == tiles - 1;
                if (!last) issue_dp();
                if (tq == 0 && uq > 0) mbar_wait<kAccFree>(base, (uq - 1) & 1, wctx, 11);
                mbar_wait<kDsReady>(base + 8 * (n & 1), (n >> 1) & 1, wctx, 12);
                tc_fence_after();
                const uint32_t a = tmem + dp_slot(q3) * kTile, db = desc_lo(base + L::kKRing + gq.s * L::kTileBytes, L::kSlab);
                static_for<8>([&](auto kk_c) {
                    constexpr int kk = decltype(kk_c)::value;
                    mma_ts_lo<packed_column(kk, kRowCols), kk * (2048 >> 4)>(leader, tm_dq, a, db, idesc_d, tq > 0 || kk > 0);
                });
                tc_commit<kKEmpty>(leader, base + 8 * gq.s);
                gq.next<L::kKStages>();
                ++n;
                q3 = q3 == 2 ? 0 : q3 + 1;
                ++tq;
                if (last) {
                    tc_commit<kAccReady>(leader, base);
                    tq = 0;
                    ++uq;
                    tiles = tiles_of(uq);
                    issue_dp();
                }
                issue_s();
            }
        } else if (warp == kRowWarps + 2) {
            // ---------------------------------------------------------------- guard
            Ring g;
            for (RowStream x(P); x.valid(); x.next(P)) {
                mbar_wait<kKFull>(base + 8 * g.s, g.phase, wctx, 13);
                const int rows = x.u.s.nk - (x.u.t0 + x.t) * kTile;
                if (rows < kTile) {
                    zero_tile_rows<HD>(base + L::kKRing + g.s * L::kTileBytes, 0, rows, lane);
                    fence_proxy_async_smem();
                }
                SA_ARRIVE(kPassed, base + 8 * g.s);
                if (lane == 0) mbar_arrive<kKEmpty>(base + 8 * g.s);
                g.next<L::kKStages>();
            }
        }
    } else {
        // -------------------------------------------------------------------- compute: a query per thread, 32 keys per group
        reg_alloc<kRowRegsCompute>();
        const int grp = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(row & ~31) << 16;
        const float2 c2 = make_float2(p.scale * kLog2e, p.scale * kLog2e);
        uint32_t n = 0, nu = 0, n3 = 0;
        for (Walk w(P, p.H); w.valid(); w.next()) {
            const RowUnit u = row_unit(P, w);
            const int i = u.i0 + row;
            const bool mine = i < u.s.nq;
            const int sees = uniform(u.i0 + u.s.off());      // last key that row 0 sees (below 0: none)
            const int64_t at = ((int64_t)u.s.b * p.H + u.h) * p.Nq + u.s.q0 + i;
            // (negated: P = exp2(S c2 + ls); a row that sees nothing, or has scores of -inf only, has P = 0.  All loads before what uses them.)
            float ls = INFINITY, dl = 0.f;
            if (mine && sees + row >= 0) {
                ls = -P.lse[at];
                dl = -P.delta[at];
            }
            const float f = F16 ? ds_factor(P, u.s.id) : p.scale;
            const float2 sc = make_float2(f, f);
            dl = ls == INFINITY ? 0.f : dl * f;
            ls = ls == INFINITY ? -INFINITY : ls * kLog2e;
            const float2 nls = make_float2(ls, ls), ndl = make_float2(dl, dl);
            const int masked_from = u.first_masked();
#pragma unroll 1
            for (int t = 0; t < u.n; ++t, ++n) {
                const uint32_t s_addr = tmem + s_slot(n3) * kTile + lanes + kRowCols * grp, dp_addr = tmem + dp_slot(n3) * kTile + lanes + kRowCols * grp;
                n3 = n3 == 2 ? 0 : n3 + 1;
                mbar_wait<kSReady>(base + 8 * (n & 1), (n >> 1) & 1, wctx, 14);
                tc_fence_after();
                float pr[kRowCols];
                tmem_ld32(s_addr, reinterpret_cast<uint32_t(&)[32]>(pr[0]));
                tmem_wait_ld();
                tc_fence_before();
                SA_ARRIVE(kSRead, base + 8 * (n & 1));
                const bool masked = t >= masked_from;
                uint32_t seen = ~0u;
                if (masked) {
                    const int hi = sees + row - (u.t0 + t) * kTile - kRowCols * grp;        // columns up to this one
                    seen = hi >= 31 ? ~0u : hi < 0 ? 0u : ~0u >> (31 - hi);
                }
#pragma unroll
                for (int c = 0; c < kRowCols; c += 2) {
                    const float2 y = __ffma2_rn(make_float2(pr[c], pr[c + 1]), c2, nls);
                    pr[c] = ex2(y.x);
                    pr[c + 1] = ex2(y.y);
                }
                mbar_wait<kDpReady>(base + 8 * (n & 1), (n >> 1) & 1, wctx, 15);
                tc_fence_after();
                uint32_t v[kRowCols], pk[kRowCols / 2];
                tmem_ld32(dp_addr, v);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < kRowCols; e += 2) {
                    float2 y = __ffma2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc, ndl);
                    y = __fmul2_rn(y, make_float2(pr[e], pr[e + 1]));
                    if (masked) {
                        y.x = (seen >> e) & 1 ? y.x : 0.f;
                        y.y = (seen >> e) & 2 ? y.y : 0.f;
                    }
                    pk[e >> 1] = E::pack(y.x, y.y);
                }
                tmem_st16(dp_addr, pk);
                tmem_wait_st();
                tc_fence_before();
                SA_ARRIVE(kDsReady, base + 8 * (n & 1));
            }
            // ---- each group writes a quarter of the columns
            if (u.n > 0) {
                mbar_wait<kAccReady>(base, nu & 1, wctx, 16);
                tc_fence_after();
                ++nu;
            }
            constexpr int kOut = HD / kRowGroups;
            const float undo = p.scale * one_over(f);
            const int col = grp * kOut;
            __nv_bfloat16* const dst = dq + u.s.b * p.dq.b + (int64_t)(u.s.q0 + i) * p.dq.n + u.h * p.dq.h + col;
            float* const part = P.part0 + (int64_t)u.split * p.B * p.H * p.Nq * HD + at * HD + col;
#pragma unroll
            for (int c0 = 0; c0 < kOut; c0 += 16) {
                uint32_t x[16];
                if (u.n > 0) {
                    tmem_ld16(tm_dq + lanes + col + c0, x);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = 0u;
                }
                if (!mine) continue;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if constexpr (F16) x[e] = __float_as_uint(__uint_as_float(x[e]) * undo);
                    x[e] = sees + row < 0 ? 0u : x[e];           // (zero, whatever the row's masked zeros met in K)
                }
                if (P.splits > 1) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) *reinterpret_cast<uint4*>(part + c0 + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e += 8)
                        if (col + c0 + e < p.D)
                            *reinterpret_cast<uint4*>(dst + c0 + e) =
                                make_uint4(E::pack(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), E::pack(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])),
                                           E::pack(__uint_as_float(x[e + 4]), __uint_as_float(x[e + 5])), E::pack(__uint_as_float(x[e + 6]), __uint_as_float(x[e + 7])));
                }
            }
            if (u.n > 0) {
                tc_fence_before();
                SA_ARRIVE(kAccFree, base);
            }
        }
    }
    if (p.cu_q != nullptr && P.splits == 1) zero_outside(dq, p.dq, p.H, p.D, p.Nq, p.cu_q, p.S, blockIdx.x, gridDim.x);
    tc_fence_before();
    __syncthreads();
    if (warp == kRowWarps) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

#undef SA_ARRIVE

// Adds the shares of a gradient in their order: [splits][B][heads][n][D] fp32 -> rows (b, i, h); a thread takes 4 columns.
template <int HD, bool F16>
__global__ void __launch_bounds__(256) causal_add_kernel(const float* __restrict__ part, __nv_bfloat16* __restrict__ out, sa_strides so, int splits, int B,
                                                        int heads, int n, int D, const int* cu, int S) {
    using E = ptx::El<F16>;
    constexpr int kRows = 256 / (HD / 4);          // of a block
    const int64_t rows = (int64_t)B * heads * n;
    const unsigned at = blockIdx.x * kRows + threadIdx.x / (HD / 4);
    const int c = (int)(threadIdx.x % (HD / 4)) * 4;
    if (at >= rows || c >= D) return;
    const unsigned bh = at / (unsigned)n;
    const int i = (int)(at - bh * (unsigned)n), h = (int)(bh % (unsigned)heads), b = (int)(bh / (unsigned)heads);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (cu == nullptr || (i >= cu[0] && i < cu[S])) {         // (rows outside every sequence: zeros)
#pragma unroll 4
        for (int x = 0; x < splits; ++x) {
            const float4 v = *reinterpret_cast<const float4*>(part + (x * rows + at) * HD + c);
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
    }
    *reinterpret_cast<uint2*>(out + b * so.b + (int64_t)i * so.n + h * so.h + c) = make_uint2(E::pack(s.x, s.y), E::pack(s.z, s.w));
}

template <int HD>
int launch_add(bool f16, const float* part, void* out, const sa_strides& so, int splits, int B, int heads, int n, int D, const int* cu, int S,
               cudaStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)B * heads * n * (HD / 4) + 255) / 256);
    if (f16) causal_add_kernel<HD, true><<<grid, 256, 0, st>>>(part, (__nv_bfloat16*)out, so, splits, B, heads, n, D, cu, S);
    else causal_add_kernel<HD, false><<<grid, 256, 0, st>>>(part, (__nv_bfloat16*)out, so, splits, B, heads, n, D, cu, S);
    host::count_launches(1);
    return cudaGetLastError() == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
}

struct BwdPlan {
    int64_t items_q, items_k;         // at most
    int splits_q, splits_k;
    int parts;                        // fp16: of a sequence, for the norms
    size_t delta, list_q, list_k, part_q, part_k, part_v, norms, bytes;
};
inline BwdPlan plan_bwd(const CParams& c, bool f16) {
    BwdPlan f{};
    const bool packed = c.cu_q != nullptr;
    f.items_q = packed ? list_capacity(c.Nq, kTile, c.S) : (int64_t)ceil_div(c.Nq, kTile) * c.S;
    f.items_k = packed ? list_capacity(c.Nk, kTile, c.S) : (int64_t)ceil_div(c.Nk, kTile) * c.S;
    const int sms = host::sm_count();
    // (a step of either kernel takes about 1.3 us at D 128, which is taken for every head dim; adding shares 5 for a tensor and the partial rows' way through memory)
    const double row_us = (double)c.B * tile_columns(c.D) * 8 / 5e6;
    const int steps_q = ceil_div(c.max_k, kTile);
    f.splits_q = plan_shares((double)f.items_q * c.H, steps_q, mean_steps(c, steps_q), sms, 16, 3.8, row_us * c.H * c.Nq / 1.3);
    const int tiles = ceil_div(c.max_q, kTile), steps_k = (int)((int64_t)tiles * c.G < (1 << 20) ? tiles * c.G : 1 << 20);
    f.splits_k = plan_shares((double)f.items_k * c.Hkv, steps_k, c.max_q == c.max_k ? mean_steps(c, tiles) * c.G : steps_k, sms, 16, 7.7,
                             2 * row_us * c.Hkv * c.Nk / 1.3);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t x = at; at += (n + 255) / 256 * 256; return x; };
    f.delta = take((size_t)c.B * c.H * c.Nq * 4);
    f.list_q = take(packed ? list_bytes(f.items_q) : 0);
    f.list_k = take(packed ? list_bytes(f.items_k) : 0);
    f.part_q = take(f.splits_q > 1 ? (size_t)f.splits_q * c.B * c.H * c.Nq * tile_columns(c.D) * 4 : 0);
    f.part_k = take(f.splits_k > 1 ? (size_t)f.splits_k * c.B * c.Hkv * c.Nk * tile_columns(c.D) * 4 : 0);
    f.part_v = take(f.splits_k > 1 ? (size_t)f.splits_k * c.B * c.Hkv * c.Nk * tile_columns(c.D) * 4 : 0);
    // (blocks that fill the multiprocessors, with a few rows a thread)
    const int64_t blocks = ((int64_t)c.B * c.H * c.Nq + (int64_t)c.B * c.Hkv * c.Nk) / (128LL * c.S) + 1;
    f.parts = (int)(blocks < kMostParts ? blocks : kMostParts);
    if (f.parts > ceil_div(8 * sms, c.S)) f.parts = ceil_div(8 * sms, c.S);
    f.norms = take(f16 ? (size_t)c.S * f.parts * sizeof(float2) : 0);
    f.bytes = at;
    return f;
}

template <int HD, bool F16>
int launch_bwd_tc(const CParams& c, const void* q, const void* k, const void* v, const void* o, const void* o_low, const float* lse, const void* d_o,
                  void* dq, void* dk, void* dv, uint8_t* ws, DeviceStatus* status, cudaStream_t st) {
    const BwdPlan f = plan_bwd(c, F16);
    if (f.items_q * c.H * f.splits_q > 0x3fffffff || f.items_k * c.Hkv * f.splits_k > 0x3fffffff) return SA_ERR_UNSUPPORTED;
    CUtensorMap mq, mk, mv, mo;
    if (!host::make_map(&mq, q, c.B, c.Nq, c.H, c.D, c.q, kTile, F16) || !host::make_map(&mk, k, c.B, c.Nk, c.Hkv, c.D, c.k, kTile, F16) ||
        !host::make_map(&mv, v, c.B, c.Nk, c.Hkv, c.D, c.v, kTile, F16) || !host::make_map(&mo, d_o, c.B, c.Nq, c.H, c.D, c.d_o, kTile, F16))
        return SA_ERR_BAD_STRIDE;
    if (!allow_dynamic_smem((const void*)causal_dkv_tc_kernel<HD, F16>, ColLayout<HD>::kBytes) ||
        !allow_dynamic_smem((const void*)causal_dq_tc_kernel<HD, F16>, RowLayout<HD>::kBytes))
        return SA_ERR_LAUNCH;
    float* delta = reinterpret_cast<float*>(ws + f.delta);
    const int64_t rows = (int64_t)c.B * c.Nq * c.H;
    constexpr int kPerBlock = 256 / (HD / 8);
    float2* const norms = reinterpret_cast<float2*>(ws + f.norms);
    const int64_t delta_blocks = (rows + kPerBlock - 1) / kPerBlock + (F16 ? (int64_t)c.S * f.parts : 0);
    if (delta_blocks > 0x7fffffff) return SA_ERR_UNSUPPORTED;
    causal_delta16_kernel<HD, F16><<<(unsigned)delta_blocks, 256, 0, st>>>(c, (const __nv_bfloat16*)o, (const __nv_bfloat16*)o_low, (const __nv_bfloat16*)v,
                                                                           (const __nv_bfloat16*)d_o, delta, norms, f.parts);
    host::count_launches(1);
    BwdParams P{};
    P.c = c;
    P.lse = lse;
    P.delta = delta;
    P.norms = norms;
    P.parts = f.parts;
    P.status = status;
    P.wait_limit_ns = host::wait_limit_ns();
    P.work.S = c.S;
    P.work.last = last_tile(kTile);
    PlanParams plan{};
    if (c.cu_q != nullptr) {
        plan.list[0] = reinterpret_cast<ListHead*>(ws + f.list_q);
        plan.list[1] = reinterpret_cast<ListHead*>(ws + f.list_k);
        plan.rows[0] = plan.rows[1] = kTile;
        plan.by_key[1] = 1;
        plan.capacity[0] = (int)f.items_q;
        plan.capacity[1] = (int)f.items_k;
        causal_plan_kernel<<<2, 1024, 0, st>>>(c, plan);
        host::count_launches(1);
    }
    const int sms = host::sm_count();
    int rc = SA_OK;
    if (dk || dv) {
        P.work.head = plan.list[1];
        P.work.tiles = ceil_div(c.Nk, kTile);
        P.work.descending = 0;
        P.splits = f.splits_k;
        P.part0 = reinterpret_cast<float*>(ws + f.part_k);
        P.part1 = reinterpret_cast<float*>(ws + f.part_v);
        const int64_t units = f.items_k * c.Hkv * f.splits_k;
        causal_dkv_tc_kernel<HD, F16><<<(unsigned)(units < sms ? units : sms), kColThreads, ColLayout<HD>::kBytes, st>>>(
            P, mq, mk, mv, mo, (__nv_bfloat16*)dk, (__nv_bfloat16*)dv);
        host::count_launches(1);
        if (f.splits_k > 1) {
            if (dk) rc = launch_add<HD>(F16, P.part0, dk, c.dk, f.splits_k, c.B, c.Hkv, c.Nk, c.D, c.cu_k, c.S, st);
            if (dv && rc == SA_OK) rc = launch_add<HD>(F16, P.part1, dv, c.dv, f.splits_k, c.B, c.Hkv, c.Nk, c.D, c.cu_k, c.S, st);
        }
    }
    if (dq && rc == SA_OK) {
        P.work.head = plan.list[0];
        P.work.tiles = ceil_div(c.Nq, kTile);
        P.work.descending = 1;
        P.splits = f.splits_q;
        P.part0 = reinterpret_cast<float*>(ws + f.part_q);
        const int64_t units = f.items_q * c.H * f.splits_q;
        causal_dq_tc_kernel<HD, F16><<<(unsigned)(units < sms ? units : sms), kRowThreads, RowLayout<HD>::kBytes, st>>>(P, mq, mk, mv, mo, (__nv_bfloat16*)dq);
        host::count_launches(1);
        if (f.splits_q > 1) rc = launch_add<HD>(F16, P.part0, dq, c.dq, f.splits_q, c.B, c.H, c.Nq, c.D, c.cu_q, c.S, st);
    }
    if (rc != SA_OK) return rc;
    return cudaGetLastError() == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
}

}  // namespace causal
}  // namespace sa
