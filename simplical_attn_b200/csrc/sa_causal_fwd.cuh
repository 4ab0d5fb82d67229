// Causal attention forward on the sm_100a tensor cores (bf16 / fp16; head dims up to 128 that are multiples of 8, in tiles of 64 or
// 128 columns that the TMA loads fill up with zeros).
//
//     S = Q K^T,  P = exp2(S scale log2e - m),  O = sum over key tiles of P V / l,  with the running maximum m and sum l per row.
//
// A unit is a pair of 128-query tiles of one head (and one share of the keys); persistent blocks, one per multiprocessor, take
// the units from the most to the least expensive in alternating direction.  Both query tiles stream through the same
// 128-key tiles of K and V.
//
// Warps.  0-3 / 4-7: softmax group of query tile 0 / 1, a row per thread, also writes the rows out.  8: MMA issuer.  9: TMA.
// 10: V guard (see below).  The query tiles work in opposite phase: while one is in its softmax the tensor cores work for the
// other.  The issuer's loop runs on over units: S of the next unit's first tile is computed while the rows are written out.
// Tensor memory: S0 | S1 (128 columns each) | O0 | O1 (D columns) | and at D = 64 P0 | P1 (64 columns of packed 16-bit values), which
// at D = 128 overwrite S.  With columns of its own for P the next S is computed as soon as the softmax has S in registers;
// at D = 128 it waits for P V.
//
// Per pair of query tiles and 128 keys at D = 128 the MMAs take 2048 cycles (128 x 128 x 16 in 64) and so do the exponentials
// (16 per clock).  Measured back to back for a second, bf16 B 2 N 8192 H 16/4: 493 us at D 128 (1116 TFLOP/s under the power cap;
// 470 with pauses; 525 where the low part of O is wanted, too), 375 us at D 64 (732 TFLOP/s).  Under a profiler at 1.60 GHz a pair
// takes about 3400 cycles at D 128, the tensor pipe is 63 % active: what is left is the chain from S through the softmax to P V of
// each query tile.  At D 64 the exponentials take 70 % of what they could.  Dropped, each against the kernel of its time: two threads
// to a row (sixteen softmax warps: 8 % slower at D 128, no difference at D 64), exponentials on the FMA pipes as well, every eighth
// to every third pair (3 to 10 % slower).
//
// Masked scores become -inf whatever they are, so P is an exact zero there; V rows of tiles with masked scores might still meet
// that zero as NaN or infinity.  The guard warp looks through those tiles before their MMAs: rows behind the sequence's
// keys become zeros, and an element that is not finite becomes a zero whose row is noted per column; the epilogue puts the
// infinity or NaN back into the rows that see it.
#pragma once

#include "sa_causal_tc.cuh"

namespace sa {
namespace causal {

constexpr int kFwdThreads = 384;
constexpr int kFwdRegsSoftmax = 208, kFwdRegsRest = 88;
static_assert(2 * kFwdRegsSoftmax + kFwdRegsRest <= 3 * 168, "register pool of the block (384 x 168 at launch)");
constexpr float kRescaleLog2 = 8.0f;      // the running maximum is kept until a score exceeds it by this much (log2)

struct FwdParams {
    CParams c;
    WorkList work;            // tiles of 128 row_tiles queries
    int row_tiles;            // query tiles of a unit: 2, or 1 where that spreads a small problem over more multiprocessors
    int splits;               // shares of the keys of a pair
    float* part_o;            // splits > 1: [splits][B H Nq][D] partial rows, and their LSE [splits][B H Nq]
    float* part_lse;
    DeviceStatus* status;
    uint64_t wait_limit_ns;
};

template <int HD>
struct FwdLayout {
    static constexpr int kSlabs = HD / 64;
    static constexpr int kSlab = kTile * 128;                    // bytes of a [128 x 64] slab
    static constexpr int kTileBytes = kSlabs * kSlab;
    static constexpr int kStages = HD == 128 ? 5 : 8;            // ring of K and V tiles
    static constexpr bool kOwnP = HD == 64;                      // P beside S in tensor memory, not over it
    static constexpr int kMisc = 384;                            // behind the barriers
    static constexpr int kBad = 512;                             // guard: [3][HD] first rows that hold +inf, -inf, NaN
    static constexpr int kQ = 2048;
    static constexpr int kRing = kQ + 2 * kTileBytes;
    static constexpr int kBytes = kRing + kStages * kTileBytes + 1024;       // 1024: alignment of the base
    static_assert(kBad + 3 * HD * 4 <= kQ && kQ % 1024 == 0 && kBytes <= 227 * 1024, "shared memory of a block");
};

// A unit: query tiles r = 0, 1 at rows i0 + 128 r take key tiles [t0, t0 + m[r]).
struct FwdUnit {
    Seq s;
    int h, split, i0, t0, m0, m1;
    __device__ __forceinline__ int m(int r) const { return r ? m1 : m0; }
    __device__ __forceinline__ int tiles() const { return max(m0, m1); }
    // first key tile (counted from t0) in which row i0 + 128 r does not see every key
    __device__ __forceinline__ int first_masked(int r) const {
        const int limit = i0 + kTile * r + s.off() + 1;           // keys that row sees
        return max((limit > 0 ? limit : 0) / kTile - t0, 0);
    }
};

struct FwdWalk {
    int u, round, count;
    __device__ __forceinline__ explicit FwdWalk(const FwdParams& P) {
        count = list_count(P.work) * P.c.H * P.splits;
        round = 0;
        u = blockIdx.x;
    }
    __device__ __forceinline__ bool valid() const { return u < count; }
    __device__ __forceinline__ void next() {
        ++round;
        u = round * (int)gridDim.x + ((round & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
    }
    __device__ __forceinline__ FwdUnit unit(const FwdParams& P) const {
        FwdUnit r;
        const int x = u / P.splits, item = x / P.c.H;
        r.split = u - x * P.splits;
        r.h = x - item * P.c.H;
        int tile;
        list_item(P.c, P.work, item, r.s, tile);
        r.i0 = tile * P.row_tiles * kTile;
        const int n0 = key_tiles(r.i0, kTile, r.s.nq, r.s.nk), n1 = P.row_tiles > 1 ? key_tiles(r.i0 + kTile, kTile, r.s.nq, r.s.nk) : 0;
        const int share = (max(n0, n1) + P.splits - 1) / P.splits;
        r.t0 = r.split * share;
        r.m0 = min(max(n0 - r.t0, 0), share);
        r.m1 = min(max(n1 - r.t0, 0), share);
        return r;
    }
};

struct Ring {
    int s = 0;
    uint32_t phase = 0;
    template <int N>
    __device__ __forceinline__ void next() {
        if (++s == N) {
            s = 0;
            phase ^= 1;
        }
    }
};

// Whether one of two packed elements is infinite or NaN.
template <bool F16>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t kExp = F16 ? 0x7c00u : 0x7f80u;
    return (~w & kExp) == 0 || (~w & (kExp << 16)) == 0;
}
// Two values as packed 16-bit ones, and what that rounding took from them.
template <bool F16>
__device__ __forceinline__ void pack_split(float a, float b, uint32_t& w, uint32_t& low) {
    using E = ptx::El<F16>;
    w = E::pack(a, b);
    low = E::pack(a - E::lo(w), b - E::hi(w));
}

template <int HD, bool F16>
__global__ void __launch_bounds__(kFwdThreads, 1)
causal_fwd_tc_kernel(const __grid_constant__ FwdParams P, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, __nv_bfloat16* __restrict__ o, __nv_bfloat16* __restrict__ o_low, float* __restrict__ lse) {
    using L = FwdLayout<HD>;
    using namespace ptx;
    using E = El<F16>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_u32(smem);
    const CParams& p = P.c;

    constexpr int kFull = 0;                          // [stage] K or V tile landed
    constexpr int kEmpty = kFull + 8 * L::kStages;    //         read by the MMAs and passed by the guard
    constexpr int kPassed = kEmpty + 8 * L::kStages;  //         looked through by the guard
    constexpr int kQFull = kPassed + 8 * L::kStages;  // [query tile] Q landed
    constexpr int kQFree = kQFull + 16;               //              the unit's last S MMAs have read it
    constexpr int kSReady = kQFree + 16;              //              S computed
    constexpr int kPReady = kSReady + 16;             //              first half of P stored
    constexpr int kP2Ready = kPReady + 16;            //              second half
    constexpr int kOReady = kP2Ready + 16;            //              O final
    constexpr int kOFree = kOReady + 16;              //              O read out
    constexpr int kSRead = kOFree + 16;               //              kOwnP: S is in registers
    constexpr int kPvDone = kSRead + 16;              //              kOwnP: P V of the tile done
    static_assert(kPvDone + 16 <= L::kMisc, "room for the barriers");
    uint32_t* tmem_slot = (uint32_t*)(smem + L::kMisc);
    volatile int* const bad_unit = (volatile int*)(smem + L::kMisc + 8);      // 1 + index of the unit the noted rows are of
    volatile int* const done = (volatile int*)(smem + L::kMisc + 16);         // [query tile] units whose rows are written out
    int* const bad = (int*)(smem + L::kBad);
    const WaitCtx wctx{base + L::kMisc + 4, P.status, P.wait_limit_ns};

    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    if (tid == 0) {
        auto init = [&](int off, int n, uint32_t count) {
            for (int x = 0; x < n; ++x) mbar_init((uint64_t*)(smem + off) + x, count);
        };
        init(kFull, L::kStages, 1);
        init(kEmpty, L::kStages, 2);
        init(kQFull, 2, 1);
        init(kQFree, 2, 1);
        init(kSReady, 2, 1);
        init(kPReady, 2, 4);
        init(kP2Ready, 2, 4);
        init(kOReady, 2, 1);
        init(kOFree, 2, 4);
        init(kSRead, 2, 4);
        init(kPvDone, 2, 1);
        init(kPassed, L::kStages, 1);
        *(volatile int*)(smem + L::kMisc + 4) = 0;
        *bad_unit = 0;
        done[0] = done[1] = 0;
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
#define SA_ARRIVE(OFF, BASE)                       \
    do {                                           \
        __syncwarp();                              \
        if (lane == 0) mbar_arrive<(OFF)>(BASE);   \
    } while (0)

    if (warp >= 8) {
        reg_dealloc<kFwdRegsRest>();
        if (warp == 9) {
            // ---------------------------------------------------------------- TMA
            if (lane == 0) {
                prefetch_tensormap(&map_q);
                prefetch_tensormap(&map_k);
                prefetch_tensormap(&map_v);
                Ring g;
                uint32_t nq[2] = {0, 0};
                for (FwdWalk w(P); w.valid(); w.next()) {
                    const FwdUnit u = w.unit(P);
                    const int hk = u.h / p.G, nt = u.tiles();
                    auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head) {
                        mbar_arrive_expect_tx(bar, L::kTileBytes);
#pragma unroll
                        for (int sl = 0; sl < L::kSlabs; ++sl) tma_load_4d(dst + sl * L::kSlab, map, bar, sl * 64, row, head, u.s.b);
                    };
                    for (int t = 0; t < nt; ++t)
#pragma unroll 1
                        for (int kv = 0; kv < 2; ++kv) {
                            mbar_wait<kEmpty>(base + 8 * g.s, g.phase ^ 1, wctx, 2 + kv);
                            load(base + L::kRing + g.s * L::kTileBytes, kv ? &map_v : &map_k, base + kFull + 8 * g.s, u.s.k0 + (u.t0 + t) * kTile, hk);
                            g.next<L::kStages>();
                            if (t == 0 && kv == 0)      // behind the first keys: those need not wait for the last unit's Q to be free
                                for (int r = 0; r < 2; ++r)
                                    if (u.m(r) > 0) {
                                        mbar_wait<kQFree>(base + 8 * r, (nq[r] & 1) ^ 1, wctx, 1);
                                        load(base + L::kQ + r * L::kTileBytes, &map_q, base + kQFull + 8 * r, u.s.q0 + u.i0 + kTile * r, u.h);
                                        ++nq[r];
                                    }
                        }
                }
            }
            __syncwarp();
        } else if (warp == 8) {
            // ---------------------------------------------------------------- MMA issuer
            const uint32_t leader = elect_one();
            const uint32_t idesc_s = make_idesc(128, kTile, false, false, F16), idesc_o = make_idesc(128, HD, false, true, F16);
            uint32_t nq0 = 0, nq1 = 0, np0 = 0, np1 = 0;       // per query tile: units with tiles, tiles so far
            auto issue_s = [&](int r, int buf, bool last) {
                const uint32_t da = desc_lo(base + L::kQ + r * L::kTileBytes, 16), db = desc_lo(base + L::kRing + buf * L::kTileBytes, 16);
                static_for<HD / 16>([&](auto kk_c) {
                    constexpr int kk = decltype(kk_c)::value, off = ((kk >> 2) * L::kSlab + (kk & 3) * 32) >> 4;
                    mma_ss_lo<off, off>(leader, tmem + r * kTile, da, db, idesc_s, kk > 0);
                });
                tc_commit<kSReady>(leader, base + 8 * r);
                if (last) tc_commit<kQFree>(leader, base + 8 * r);
            };
            // S of a unit's first key tile, for both query tiles
            auto first_s = [&](const FwdUnit& u, const Ring& g) {
                if (u.tiles() == 0) return;
                mbar_wait<kFull>(base + 8 * g.s, g.phase, wctx, 4);
                auto one = [&](int r, int m, uint32_t nq, uint32_t np) {
                    if (m == 0) return;
                    if (L::kOwnP && np > 0) mbar_wait<kSRead>(base + 8 * r, (np - 1) & 1, wctx, 16);
                    mbar_wait<kQFull>(base + 8 * r, nq & 1, wctx, 5);
                    tc_fence_after();
                    issue_s(r, g.s, m == 1);
                };
                one(0, u.m0, nq0, np0);
                one(1, u.m1, nq1, np1);
                tc_commit<kEmpty>(leader, base + 8 * g.s);
            };
            Ring g;
            FwdWalk w(P);
            make_uniform(w.count);
            // (of a unit the issuer only uses its counts of tiles)
            auto unit = [&] {
                FwdUnit x = w.unit(P);
                make_uniform(x.m0);
                make_uniform(x.m1);
                x.t0 = uniform(x.first_masked(0));          // the first tile to wait for the guard at
                return x;
            };
            FwdUnit u;
            if (w.valid()) {
                u = unit();
                first_s(u, g);
            }
            while (w.valid()) {
                w.next();
                FwdUnit un = u;
                if (w.valid()) un = unit();
                const int nt = u.tiles(), guarded = u.t0;
#pragma unroll 1
                for (int t = 0; t < nt; ++t) {
                    g.next<L::kStages>();
                    const Ring v = g;
                    Ring k = g;
                    k.next<L::kStages>();
                    const uint32_t db = desc_lo(base + L::kRing + v.s * L::kTileBytes, L::kSlab);
                    mbar_wait<kFull>(base + 8 * v.s, v.phase, wctx, 6);
                    if (t >= guarded) mbar_wait<kPassed>(base + 8 * v.s, v.phase, wctx, 7);
                    // (the query tile as a constant: counters indexed by it would lie in memory)
                    auto one = [&](auto r_c, int m, uint32_t& nq, uint32_t& np) {
                        constexpr int r = decltype(r_c)::value;
                        if (t >= m) return;
                        const uint32_t rb = base + 8 * r, tm_o = tmem + 2 * kTile + r * HD;
                        const uint32_t tm_p = L::kOwnP ? tmem + 2 * kTile + 2 * HD + r * (kTile / 2) : tmem + r * kTile;
                        auto next_s = [&] {
                            mbar_wait<kFull>(base + 8 * k.s, k.phase, wctx, 11);
                            if (L::kOwnP) mbar_wait<kSRead>(rb, np & 1, wctx, 16);
                            tc_fence_after();
                            issue_s(r, k.s, t + 1 == m - 1);
                        };
                        if (L::kOwnP && t + 1 < m) next_s();
                        if (t == 0 && nq > 0) mbar_wait<kOFree>(rb, (nq - 1) & 1, wctx, 8);
                        mbar_wait<kPReady>(rb, np & 1, wctx, 9);
                        tc_fence_after();
                        static_for<4>([&](auto kk_c) {
                            constexpr int kk = decltype(kk_c)::value;
                            mma_ts_lo<kk * 8, kk * (2048 >> 4)>(leader, tm_o, tm_p, db, idesc_o, t > 0 || kk > 0);
                        });
                        mbar_wait<kP2Ready>(rb, np & 1, wctx, 10);
                        tc_fence_after();
                        static_for<4>([&](auto kk_c) {
                            constexpr int kk = decltype(kk_c)::value + 4;
                            mma_ts_lo<kk * 8, kk * (2048 >> 4)>(leader, tm_o, tm_p, db, idesc_o, true);
                        });
                        if (L::kOwnP) tc_commit<kPvDone>(leader, rb);
                        if (t == m - 1) {
                            tc_commit<kOReady>(leader, rb);
                            ++nq;
                        } else if (!L::kOwnP) {
                            next_s();
                        }
                        ++np;
                    };
                    one(std::integral_constant<int, 0>{}, u.m0, nq0, np0);
                    one(std::integral_constant<int, 1>{}, u.m1, nq1, np1);
                    tc_commit<kEmpty>(leader, base + 8 * v.s);
                    g.next<L::kStages>();
                    if (t + 1 < nt) tc_commit<kEmpty>(leader, base + 8 * k.s);
                }
                u = un;
                if (w.valid()) first_s(u, g);
            }
        } else if (warp == 10) {
            // ---------------------------------------------------------------- V guard
            // 8 elements at `at`, of row j and columns d0.., of which this lane's are not all finite if `any`
            auto note = [&](bool any, uint32_t at, const uint4& x, int j, int d0, uint32_t units) {
                constexpr uint32_t kExp = F16 ? 0x7c00u : 0x7f80u;
                if (*bad_unit != (int)units + 1) {
                    // what is noted now may still be wanted by rows of earlier units: they are written out first
                    auto written = [&] { return done[0] >= (int)units && done[1] >= (int)units; };
                    if (!__all_sync(0xffffffffu, mbar_wait_on(written, written, wctx, 18))) return;
                    for (int d = lane; d < 3 * HD; d += 32) bad[d] = 0x7fffffff;
                    __threadfence_block();
                    __syncwarp();
                    if (lane == 0) *bad_unit = (int)units + 1;
                    __syncwarp();
                }
                if (any) {
                    uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t h = (word[e >> 1] >> (16 * (e & 1))) & 0xffffu;
                        if ((~h & kExp) != 0) continue;
                        atomicMin(&bad[((h & (0x7fffu ^ kExp)) != 0 ? 2 : (int)(h >> 15)) * HD + d0 + e], j);
                        word[e >> 1] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
                    }
                    sts128(at, make_uint4(word[0], word[1], word[2], word[3]));
                }
                __threadfence_block();
                __syncwarp();
            };
            Ring g;
            uint32_t units = 0;
            for (FwdWalk w(P); w.valid(); w.next(), ++units) {
                const FwdUnit u = w.unit(P);
                const int nt = u.tiles(), guarded = u.first_masked(0);
                for (int t = 0; t < nt; ++t) {
                    // (the guard takes part in every phase of the ring, so that it is never a turn behind or ahead)
                    mbar_wait<kFull>(base + 8 * g.s, g.phase, wctx, 12);       // K
                    SA_ARRIVE(kPassed, base + 8 * g.s);
                    if (lane == 0) mbar_arrive<kEmpty>(base + 8 * g.s);
                    g.next<L::kStages>();
                    mbar_wait<kFull>(base + 8 * g.s, g.phase, wctx, 13);       // V
                    if (t >= guarded) {
                        const uint32_t tile = base + L::kRing + g.s * L::kTileBytes;
                        const int j0 = (u.t0 + t) * kTile, rows = u.s.nk - j0;
                        constexpr uint32_t kExp2 = F16 ? 0x7c007c00u : 0x7f807f80u, kOne2 = F16 ? 0x04000400u : 0x00800080u;
                        // A lane takes every 32nd 16-byte chunk; the chunks of a slab's 128-byte row are XOR-ed with row & 7.  First only
                        // whether there is anything to note: an exponent of ones carries into its element's sign bit.
                        uint32_t carry = 0;
#pragma unroll 8
                        for (int c = lane; c < kTile * HD / 8; c += 32) {
                            const uint4 x = lds128(tile + c * 16);
                            carry |= ((x.x & kExp2) + kOne2) | ((x.y & kExp2) + kOne2) | ((x.z & kExp2) + kOne2) | ((x.w & kExp2) + kOne2);
                        }
                        if (__any_sync(0xffffffffu, (carry & 0x80008000u) != 0))
                            for (int c = lane; c < kTile * HD / 8; c += 32) {
                                const int sl = c / (kTile * 8), row = c / 8 % kTile;
                                const uint32_t at = tile + c * 16;
                                const uint4 x = lds128(at);
                                const bool any = row < rows && (not_finite2<F16>(x.x) || not_finite2<F16>(x.y) || not_finite2<F16>(x.z) || not_finite2<F16>(x.w));
                                if (__any_sync(0xffffffffu, any)) note(any, at, x, j0 + row, sl * 64 + (((c & 7) ^ (row & 7)) << 3), units);
                            }
                        if (rows < kTile)
                            for (int c = lane; c < kTile * HD / 8; c += 32)
                                if (c / 8 % kTile >= rows) sts128(tile + c * 16, make_uint4(0, 0, 0, 0));
                        fence_proxy_async_smem();
                    }
                    SA_ARRIVE(kPassed, base + 8 * g.s);
                    if (lane == 0) mbar_arrive<kEmpty>(base + 8 * g.s);
                    g.next<L::kStages>();
                }
            }
        }
    } else {
        // -------------------------------------------------------------------- softmax groups
        reg_alloc<kFwdRegsSoftmax>();
        const int r = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(row & ~31) << 16;
        const uint32_t s_addr = tmem + r * kTile + lanes, o_addr = tmem + 2 * kTile + r * HD + lanes;
        const uint32_t p_addr = L::kOwnP ? tmem + 2 * kTile + 2 * HD + r * (kTile / 2) + lanes : s_addr;
        const uint32_t rb = base + 8 * r;
        const float c2 = p.scale * kLog2e;
        uint32_t n = 0, nu = 0, units = 0;
        for (FwdWalk w(P); w.valid(); w.next(), ++units) {
            const FwdUnit u = w.unit(P);
            const int i = u.i0 + kTile * r + row, mt = u.m(r);
            const int see = i + u.s.off() - u.t0 * kTile;            // last key the row sees, from the first of this share
            const int masked_from = u.first_masked(r);
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int t = 0; t < mt; ++t, ++n) {
                mbar_wait<kSReady>(rb, n & 1, wctx, 14);
                tc_fence_after();
                uint32_t v[kTile];
                {
                    auto ld = [&](int c) { tmem_ld32(s_addr + 32 * c, reinterpret_cast<uint32_t(&)[32]>(v[32 * c])); };
                    ld(0);
                    ld(1);
                    ld(2);
                    ld(3);
                    tmem_wait_ld();
                    if (L::kOwnP) {
                        tc_fence_before();
                        SA_ARRIVE(kSRead, rb);
                    }
                }
                if (t >= masked_from) {
                    const int hi = see - t * kTile;
#pragma unroll
                    for (int c = 0; c < kTile; c += 32) {
                        const int z = hi - c;
                        const uint32_t bits = z >= 31 ? ~0u : z < 0 ? 0u : ~0u >> (31 - z);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[c + e] = (bits & (1u << e)) ? v[c + e] : 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < kTile; e += 8)
#pragma unroll
                    for (int y = 0; y < 4; ++y) mx[y] = max3(mx[y], __uint_as_float(v[e + y]), __uint_as_float(v[e + 4 + y]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c2;
                // The running maximum moves only when it has to; then l and O are scaled down.  (O is at rest, and the columns of P are
                // free: the last tile's P V is done.  Without kOwnP this tile's S was issued behind it.)
                if (L::kOwnP && n > 0) {
                    mbar_wait<kPvDone>(rb, (n - 1) & 1, wctx, 17);
                    tc_fence_after();
                }
                float factor = 1.f;
                if (top > m + kRescaleLog2 || m == -INFINITY) {
                    if (m > -INFINITY) factor = ex2(m - top);
                    l *= factor;
                    m = top;
                }
                if (__any_sync(0xffffffffu, factor != 1.f)) {
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 16) {
                        uint32_t x[16];
                        tmem_ld16(o_addr + c0, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * factor);
                        tmem_st16(o_addr + c0, x);
                    }
                }
                const float nms = m == -INFINITY ? 0.f : -m;
                const float2 c2v = make_float2(c2, c2), nm = make_float2(nms, nms);
                float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 y = __ffma2_rn(make_float2(__uint_as_float(v[c + e]), __uint_as_float(v[c + e + 1])), c2v, nm);
                        const float2 pe = make_float2(ex2(y.x), ex2(y.y));
                        ls[(e >> 1) & 1] = __fadd2_rn(ls[(e >> 1) & 1], pe);
                        pk[e >> 1] = E::pack(pe.x, pe.y);
                    }
                    tmem_st16(p_addr + c / 2, pk);
                    if (c == kTile / 2 - 32) {
                        tmem_wait_st();
                        tc_fence_before();
                        SA_ARRIVE(kPReady, rb);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                SA_ARRIVE(kP2Ready, rb);
                l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
            }
            // ---- the rows of this unit
            const bool mine = r < P.row_tiles && i < u.s.nq;
            const int64_t at = ((int64_t)u.s.b * p.H + u.h) * p.Nq + u.s.q0 + i;
            const int64_t rows = (int64_t)p.B * p.H * p.Nq;
            const bool none = see < 0 || mt == 0 || l == 0.f;        // no key (of this share), or all scores are -inf
            if (mt > 0) {
                mbar_wait<kOReady>(rb, nu & 1, wctx, 15);
                tc_fence_after();
                ++nu;
            }
            const float inv = none ? 0.f : 1.f / l;
            const bool noted = *bad_unit == (int)units + 1;
            const int64_t out_at = u.s.b * p.o.b + (int64_t)(u.s.q0 + i) * p.o.n + u.h * p.o.h;
            float* const part = P.splits > 1 ? P.part_o + ((int64_t)u.split * rows + at) * HD : nullptr;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t x[32];
                if (mt > 0) {
                    tmem_ld32(o_addr + c0, x);
                    tmem_wait_ld();
                }
                if (c0 == HD - 32 && mt > 0) {
                    tc_fence_before();
                    SA_ARRIVE(kOFree, rb);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = none ? 0u : __float_as_uint(__uint_as_float(x[e]) * inv);
                if (noted && !none) {
                    const int limit = i + u.s.off();
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const bool up = bad[c0 + e] <= limit, down = bad[HD + c0 + e] <= limit, nan = bad[2 * HD + c0 + e] <= limit;
                        // (added: a row that is NaN or the other infinity already, through earlier keys or Q, becomes or stays NaN)
                        if (up || down || nan)
                            x[e] = __float_as_uint(__uint_as_float(x[e]) + __uint_as_float(nan || (up && down) ? 0x7fc00000u : up ? 0x7f800000u : 0xff800000u));
                    }
                }
                if (mine) {
                    if (part) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(part + c0 + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (c0 + e >= p.D) break;
                            uint32_t w[4], lo[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) pack_split<F16>(__uint_as_float(x[e + 2 * y]), __uint_as_float(x[e + 2 * y + 1]), w[y], lo[y]);
                            *reinterpret_cast<uint4*>(o + out_at + c0 + e) = make_uint4(w[0], w[1], w[2], w[3]);
                            if (o_low) *reinterpret_cast<uint4*>(o_low + out_at + c0 + e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                    }
                }
            }
            if (mine) {
                const float ll = none ? -INFINITY : (m + log2f(l)) * kLn2;
                if (part) P.part_lse[(int64_t)u.split * rows + at] = ll;
                else lse[at] = ll;
            }
            named_barrier_sync(1 + r, 128);                          // every row has looked at what the guard noted
            if (row == 0) done[r] = (int)units + 1;
        }
    }
    if (p.cu_q != nullptr) {
        zero_outside(o, p.o, p.H, p.D, p.Nq, p.cu_q, p.S, blockIdx.x, gridDim.x);
        empty_lse_outside(lse, p.H, p.Nq, p.cu_q, p.S, blockIdx.x, gridDim.x);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

#undef SA_ARRIVE

// Joins the shares of a row: O = sum_s e^(lse_s - lse) O_s.  `team` warps to a row and head, each with every team-th share; one
// warp alone would wait for its chain of loads (17 us for 28 shares of 512 rows; a team of 8: 4 us).  A share without keys has
// LSE -inf, and its row need not be written.
template <int HD, bool F16>
__global__ void __launch_bounds__(256) causal_join_kernel(const CParams p, int splits, int team, const float* __restrict__ part_o,
                                                         const float* __restrict__ part_lse, __nv_bfloat16* __restrict__ o, __nv_bfloat16* __restrict__ o_low,
                                                         float* __restrict__ lse) {
    constexpr int kPer = HD / 32;
    __shared__ float sums[8][HD + 1];
    ptx::griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, member = warp % team;
    const int64_t rows = (int64_t)p.B * p.H * p.Nq, at = (int64_t)blockIdx.x * (8 / team) + warp / team;
    const unsigned bh = (unsigned)at / (unsigned)p.Nq;          // (rows fit 31 bits)
    const int n = (int)((unsigned)at - bh * (unsigned)p.Nq), h = (int)(bh % (unsigned)p.H), b = (int)(bh / (unsigned)p.H);
    // (rows outside the sequences are written where the shares are)
    const bool in = at < rows && (p.cu_q == nullptr || (n >= p.cu_q[0] && n < p.cu_q[p.S]));
    float top = -INFINITY, sum = 0.f, acc[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
    if (in) {
        for (int s = lane; s < splits; s += 32) top = fmaxf(top, part_lse[s * rows + at]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
        for (int s = member; s < splits; s += team) {
            const float ls = part_lse[s * rows + at];
            const float* src = part_o + (s * rows + at) * HD + kPer * lane;
            float x[kPer];
#pragma unroll
            for (int e = 0; e < kPer; e += 2) {
                const float2 y = *reinterpret_cast<const float2*>(src + e);
                x[e] = y.x;
                x[e + 1] = y.y;
            }
            const float w = expf(ls - base);
            sum += w;
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] = ls == -INFINITY ? acc[e] : fmaf(w, x[e], acc[e]);
        }
    }
    if (team > 1) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) sums[warp][kPer * lane + e] = acc[e];
        if (lane == 0) sums[warp][HD] = sum;
        __syncthreads();
        if (member != 0) return;
        for (int y = 1; y < team; ++y) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] += sums[warp + y][kPer * lane + e];
            sum += sums[warp + y][HD];
        }
    }
    if (!in) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t dst = b * p.o.b + (int64_t)n * p.o.n + h * p.o.h + kPer * lane;
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
        if (kPer * lane + e >= p.D) break;
        uint32_t w, low;
        pack_split<F16>(acc[e] * inv, acc[e + 1] * inv, w, low);
        *reinterpret_cast<uint32_t*>(o + dst + e) = w;
        if (o_low) *reinterpret_cast<uint32_t*>(o_low + dst + e) = low;
    }
    if (lane == 0) lse[at] = sum == 0.f ? -INFINITY : top + logf(sum);
}

// Launches a kernel that may start while the one before it in the stream still runs (it waits for it by itself).
template <typename... Args, typename... Given>
cudaError_t launch_behind(void (*kern)(Args...), unsigned grid, unsigned block, int smem, cudaStream_t st, Given... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, Args(args)...);
}

template <int HD>
int launch_join(const CParams& p, bool f16, int splits, const float* part_o, const float* part_lse, void* o, void* o_low, float* lse, cudaStream_t st) {
    const int team = splits >= 24 ? 8 : splits >= 12 ? 4 : splits >= 4 ? 2 : 1, rows = 8 / team;
    const unsigned grid = (unsigned)(((int64_t)p.B * p.H * p.Nq + rows - 1) / rows);
    const cudaError_t e = f16 ? launch_behind(causal_join_kernel<HD, true>, grid, 256, 0, st, p, splits, team, part_o, part_lse, (__nv_bfloat16*)o,
                                            (__nv_bfloat16*)o_low, lse)
                              : launch_behind(causal_join_kernel<HD, false>, grid, 256, 0, st, p, splits, team, part_o, part_lse, (__nv_bfloat16*)o,
                                            (__nv_bfloat16*)o_low, lse);
    host::count_launches(1);
    return e == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
}

// How a call is cut up, and its workspace.
struct FwdPlan {
    int row_tiles, splits;
    int64_t items;                    // at most
    size_t list, part_o, part_lse, bytes;
};
inline FwdPlan plan_fwd(const CParams& c) {
    FwdPlan f{};
    const int sms = host::sm_count();
    auto items = [&](int tiles) {
        return c.cu_q != nullptr ? list_capacity(c.Nq, kTile * tiles, c.S) : (int64_t)ceil_div(c.Nq, kTile * tiles) * c.S;
    };
    // A key tile takes a pair of query tiles 1.95 us and a single one 1.75 (measured at D 128 and taken for every head dim, though at
    // D 64 a pair takes 1.6; nothing overlaps a single one's softmax); joining shares
    // takes 8 us and the partial rows' way through memory.
    const int tiles = ceil_div(c.max_k, kTile);
    const double mean = mean_steps(c, tiles), each = (double)c.B * c.H * c.Nq * tile_columns(c.D) * 8 / 5e6;
    double best = 1e30;
    for (int rt = 2; rt >= 1; --rt) {
        const double units = (double)items(rt) * c.H, step = rt == 2 ? 1.95 : 1.75;
        const int s = plan_shares(units, tiles, mean, sms, 32, 8.0 / step, each / step);
        const double us = walk_steps(units, tiles, mean, s, sms) * step + (s > 1 ? 8.0 + each * s : 0.0);
        if (us < best) {
            best = us;
            f.row_tiles = rt;
            f.splits = s;
        }
    }
    f.items = items(f.row_tiles);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t x = at; at += (n + 255) / 256 * 256; return x; };
    f.list = take(c.cu_q != nullptr ? list_bytes(f.items) : 0);
    const size_t rows = (size_t)c.B * c.H * c.Nq;
    f.part_o = take(f.splits > 1 ? (size_t)f.splits * rows * tile_columns(c.D) * 4 : 0);
    f.part_lse = take(f.splits > 1 ? (size_t)f.splits * rows * 4 : 0);
    f.bytes = at;
    return f;
}

template <int HD, bool F16>
int launch_fwd_tc(const CParams& c, const void* q, const void* k, const void* v, void* o, void* o_low, float* lse, uint8_t* ws, DeviceStatus* status,
                  cudaStream_t st) {
    const FwdPlan f = plan_fwd(c);
    if (f.items * c.H * f.splits > 0x3fffffff) return SA_ERR_UNSUPPORTED;
    CUtensorMap mq, mk, mv;
    if (!host::make_map(&mq, q, c.B, c.Nq, c.H, c.D, c.q, kTile, F16) || !host::make_map(&mk, k, c.B, c.Nk, c.Hkv, c.D, c.k, kTile, F16) ||
        !host::make_map(&mv, v, c.B, c.Nk, c.Hkv, c.D, c.v, kTile, F16))
        return SA_ERR_BAD_STRIDE;
    FwdParams P{};
    P.c = c;
    P.row_tiles = f.row_tiles;
    P.splits = f.splits;
    P.part_o = reinterpret_cast<float*>(ws + f.part_o);
    P.part_lse = reinterpret_cast<float*>(ws + f.part_lse);
    P.status = status;
    P.wait_limit_ns = host::wait_limit_ns();
    P.work.last = last_tile(kTile * f.row_tiles);
    P.work.tiles = ceil_div(c.Nq, kTile * f.row_tiles);
    P.work.S = c.S;
    P.work.descending = 1;
    auto kern = causal_fwd_tc_kernel<HD, F16>;
    if (!allow_dynamic_smem((const void*)kern, FwdLayout<HD>::kBytes)) return SA_ERR_LAUNCH;
    if (c.cu_q != nullptr) {
        PlanParams plan{};
        plan.list[0] = reinterpret_cast<ListHead*>(ws + f.list);
        plan.rows[0] = kTile * f.row_tiles;
        plan.capacity[0] = (int)f.items;
        P.work.head = plan.list[0];
        causal_plan_kernel<<<1, 1024, 0, st>>>(c, plan);
        host::count_launches(1);
    }
    const int64_t units = f.items * c.H * f.splits;
    const unsigned grid = (unsigned)(units < host::sm_count() ? units : host::sm_count());
    kern<<<grid, kFwdThreads, FwdLayout<HD>::kBytes, st>>>(P, mq, mk, mv, (__nv_bfloat16*)o, (__nv_bfloat16*)o_low, lse);
    host::count_launches(1);
    if (cudaGetLastError() != cudaSuccess) return SA_ERR_LAUNCH;
    return f.splits > 1 ? launch_join<HD>(c, F16, f.splits, P.part_o, P.part_lse, o, o_low, lse, st) : SA_OK;
}

}  // namespace causal
}  // namespace sa
