// Causal attention of a few queries over many keys (single tokens, a handful of drafted ones), bf16 / fp16, head dims up to
// 128 that are multiples of 8 (tiles of 64 or 128 columns, filled up with zeros).
//
// K and V are read once and little is computed with them: HBM bandwidth bounds it, latency where they are short.  The rows of
// a block are the queries of all heads that share a KV head (query i, head g of the group: row i G + g), 16 or 32 of them, so a
// key is read once for the group.  The keys of a sequence are cut into shares, a block each.  Up to eight shares are a cluster of
// blocks and join in each other's shared memory; more are joined by causal_join_kernel.
//
// The products are 16 x 8 x 16 register MMAs (mma.sync): tcgen05 works on 128 rows, of which these calls would fill 16.  A warp
// has its own 16 of every 64 keys, copied by its own asynchronous copies into its own part of shared memory, with its own
// running maximum, sum and rows of O: warps wait for nobody until they are merged at the end.
//
// Measured: 64 sequences of one token over 4096 keys, H 32/8, D 128: 164 us, 6.5 TB/s; 16 over 8192, H 32/2: 28.5 us in a graph;
// one over 2001, H 16/4, D 64: 6.6 us in a graph.  Sequences of different lengths leave the last round of blocks part empty: 16 of
// 2 to 16 K keys 42 us, 3.4 TB/s.
#pragma once

#include "sa_causal_fwd.cuh"

namespace sa {
namespace causal {

constexpr int kFewThreads = 128;
constexpr int kFewKeys = 64;              // keys of a step of the block: 16 per warp
constexpr int kFewCluster = 8;            // blocks of a cluster, at most
constexpr int kFewRowsMost = 32;          // rows (queries times heads of a group) that these kernels are taken for

struct FewParams {
    CParams c;
    int shares, row_blocks;               // of a sequence's keys, and of its rows
    int steps;                            // steps of a share, at least
    int cluster;                          // whether the shares of a sequence and head are one cluster
    float* part_o;                        // shares > 1: as in FwdParams
    float* part_lse;
};

template <int HD, int MT>
struct FewLayout {
    static constexpr int kStages = 3;
    static constexpr int kHalf = 16 * HD * 2;                       // 16 rows of K, or of V
    static constexpr int kWarp = kStages * 2 * kHalf;
    static constexpr int kQ = 16 * MT * HD * 2;
    static constexpr int kStats = 2 * 5 * 16 * MT * 4;              // m, l: [warp, block][row]
    static constexpr int kBytes = kQ + kStats + 4 * kWarp;
    static_assert(5 * 16 * MT * HD * 4 <= 4 * kWarp, "the rows of the warps are merged where K and V were, the block's behind them");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two packed elements, zeros for those that are not finite.
template <bool F16>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
    constexpr uint32_t kExp = F16 ? 0x7c00u : 0x7f80u;
    if ((~w & kExp) == 0) w &= 0xffff0000u;
    if ((~w & (kExp << 16)) == 0) w &= 0xffffu;
    return w;
}

// The blocks of a cluster: all of them here, and another's shared memory.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t of_rank(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <int HD, bool F16, int MT>
__global__ void __launch_bounds__(kFewThreads, 2)
causal_few_kernel(const __grid_constant__ FewParams P, const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k,
                  const __nv_bfloat16* __restrict__ v, __nv_bfloat16* __restrict__ o, __nv_bfloat16* __restrict__ o_low, float* __restrict__ lse) {
    using L = FewLayout<HD, MT>;
    using E = ptx::El<F16>;
    constexpr int kChunks = HD / 8;               // 16-byte chunks of a row
    extern __shared__ uint4 smem16[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>(smem16);
    const CParams& p = P.c;
    ptx::griddep_launch();                        // (the joining kernel waits for this one's end by itself)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // the shares of a sequence and head lie side by side: what runs at a time spreads over sequences of all lengths
    int x = blockIdx.x;
    const int share = x % P.shares;
    x /= P.shares;
    const int rb0 = x % P.row_blocks;
    x /= P.row_blocks;
    const int hk = x % p.Hkv;
    const Seq s = seq_of(p, x / p.Hkv);
    const int R = s.nq * p.G;
    const int64_t rows_all = (int64_t)p.B * p.H * p.Nq;
    // equal shares for sequences of all lengths: short ones have fewer (and one longer than max_k said has longer ones)
    const int steps_all = (s.nk + kFewKeys - 1) / kFewKeys, per = max(P.steps, (steps_all + P.shares - 1) / P.shares);
    const int c0 = min(min(share * per, steps_all) * kFewKeys, s.nk), c1 = min(c0 + per * kFewKeys, s.nk);
    const int steps = (c1 - c0 + kFewKeys - 1) / kFewKeys;

    const uint32_t q_st = ptx::smem_u32(smem), w_st = q_st + L::kQ + L::kStats + warp * L::kWarp;
    float* const stat_m = reinterpret_cast<float*>(smem + L::kQ);
    float* const stat_l = stat_m + 5 * 16 * MT;
    const __nv_bfloat16* const kh = k + s.b * p.k.b + (int64_t)s.k0 * p.k.n + hk * p.k.h;
    const __nv_bfloat16* const vh = v + s.b * p.v.b + (int64_t)s.k0 * p.v.n + hk * p.v.h;
    const float c2 = p.scale * kLog2e;

    for (int rb = rb0; rb * 16 * MT < R; rb += P.row_blocks) {
        const int r0 = rb * 16 * MT;
        auto load = [&](int t) {
            if (t < steps) {
                const int j0 = c0 + t * kFewKeys + warp * 16;
                const uint32_t st = w_st + (t % L::kStages) * 2 * L::kHalf;
#pragma unroll
                for (int e = 0; e < 16 * kChunks / 32; ++e) {
                    const int c = lane + 32 * e, row = c / kChunks, ch = c % kChunks, j = j0 + row;
                    const uint32_t at = st + row * HD * 2 + ((ch ^ (row & 7)) << 4);
                    const bool in = j < c1 && ch * 8 < p.D;
                    const int64_t jj = in ? j : c0, cc = in ? ch * 8 : 0;
                    cp16(at, kh + jj * p.k.n + cc, in);                   // rows behind the share: zeros
                    cp16(at + L::kHalf, vh + jj * p.v.n + cc, in);
                }
            }
            cp_commit();
        };
        if (steps > 0) {
#pragma unroll
            for (int t = 0; t < L::kStages - 1; ++t) load(t);
        }
        // rows of Q: zeros where there are none
        for (int c = tid; c < 16 * MT * kChunks; c += kFewThreads) {
            const int row = c / kChunks, ch = c % kChunks, rho = r0 + row;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (rho < R && ch * 8 < p.D) {
                const int i = rho / p.G, g = rho - i * p.G;
                w = *reinterpret_cast<const uint4*>(q + s.b * p.q.b + (int64_t)(s.q0 + i) * p.q.n + (hk * p.G + g) * p.q.h + ch * 8);
            }
            *reinterpret_cast<uint4*>(smem + row * HD * 2 + ((ch ^ (row & 7)) << 4)) = w;
        }
        __syncthreads();
        // this thread's rows (lane / 4 and 8 further down, of every 16): last key seen, running maximum and sum
        int last[2 * MT];
        float m[2 * MT], l[2 * MT], acc[MT][HD / 8][4];
#pragma unroll
        for (int y = 0; y < 2 * MT; ++y) {
            const int rho = r0 + 8 * y + (lane >> 2);
            last[y] = rho < R ? min(rho / p.G + s.off(), c1 - 1) : -1;
            m[y] = -INFINITY;
            l[y] = 0.f;
        }
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int d = 0; d < HD / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[a][d][e] = 0.f;
        const int first_last = r0 / p.G + s.off();                 // last key the block's first row sees

#pragma unroll 1
        for (int t = 0; t < steps; ++t) {
            cp_wait<L::kStages - 2>();
            __syncwarp();
            load(t + L::kStages - 1);              // (into the buffer of step t - 1, which every lane has left)
            const int j0 = c0 + t * kFewKeys + warp * 16;
            if (j0 >= c1) continue;
            const uint32_t st = w_st + (t % L::kStages) * 2 * L::kHalf;
            const bool masked = j0 + 15 > min(first_last, c1 - 1);
            uint32_t pa[MT][4];
            float sc[MT][2][4];
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int e = 0; e < 8; ++e) sc[a][e >> 2][e & 3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                uint32_t kb[4];
                {
                    const int row = (lane >> 4) * 8 + (lane & 7), ch = 2 * kk + ((lane >> 3) & 1);
                    ldm4(kb, st + row * HD * 2 + ((ch ^ (row & 7)) << 4));
                }
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    uint32_t qa[4];
                    const int row = 16 * a + (lane & 15), ch = 2 * kk + (lane >> 4);
                    ldm4(qa, q_st + row * HD * 2 + ((ch ^ (row & 7)) << 4));
                    mma16816<F16>(sc[a][0], qa, kb[0], kb[1]);
                    mma16816<F16>(sc[a][1], qa, kb[2], kb[3]);
                }
            }
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int hf = (e >> 1) & 1, j = j0 + 8 * (e >> 2) + 2 * (lane & 3) + (e & 1);
                    float& y = sc[a][e >> 2][e & 3];
                    y = !masked || j <= last[2 * a + hf] ? y * c2 : -INFINITY;
                    top[hf] = fmaxf(top[hf], y);
                }
                float f[2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float& mm = m[2 * a + hf];
                    top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 1));
                    top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 2));
                    f[hf] = 1.f;
                    if (top[hf] > mm + kRescaleLog2 || mm == -INFINITY) {
                        if (mm > -INFINITY) f[hf] = ptx::ex2(mm - top[hf]);
                        mm = top[hf];
                    }
                    l[2 * a + hf] *= f[hf];
                }
                if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                    for (int d = 0; d < HD / 8; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[a][d][e] *= f[e >> 1];
                }
                const float b0 = m[2 * a] == -INFINITY ? 0.f : m[2 * a], b1 = m[2 * a + 1] == -INFINITY ? 0.f : m[2 * a + 1];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float& y = sc[a][e >> 2][e & 3];
                    y = ptx::ex2(y - ((e >> 1) & 1 ? b1 : b0));
                    l[2 * a + ((e >> 1) & 1)] += y;
                }
                // the accumulators' layout is that of the A operand of the next product
                pa[a][0] = E::pack(sc[a][0][0], sc[a][0][1]);
                pa[a][1] = E::pack(sc[a][0][2], sc[a][0][3]);
                pa[a][2] = E::pack(sc[a][1][0], sc[a][1][1]);
                pa[a][3] = E::pack(sc[a][1][2], sc[a][1][3]);
            }
            bool odd = false;                      // a V element that is not finite, under a mask
            if (masked) {
#pragma unroll
                for (int e = 0; e < 16 * kChunks / 32; ++e) {
                    const uint4 w = ptx::lds128(st + L::kHalf + (lane + 32 * e) * 16);
                    odd |= not_finite2<F16>(w.x) || not_finite2<F16>(w.y) || not_finite2<F16>(w.z) || not_finite2<F16>(w.w);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (odd) {
                // into rows that see them key by key (a masked zero times them would not be zero), then zeros in their place
#pragma unroll 1
                for (int j = 0; j < 16; ++j)
#pragma unroll
                    for (int a = 0; a < MT; ++a)
#pragma unroll
                        for (int d = 0; d < HD / 8; ++d) {
                            const uint32_t w = ptx::lds32(st + L::kHalf + j * HD * 2 + ((d ^ (j & 7)) << 4) + (lane & 3) * 4);
                            if (!not_finite2<F16>(w)) continue;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float x = e & 1 ? E::hi(w) : E::lo(w);
                                if (!(fabsf(x) < INFINITY) && j0 + j <= last[2 * a + (e >> 1)]) acc[a][d][e] += x;
                            }
                        }
                __syncwarp();
#pragma unroll 1
                for (int e = 0; e < 16 * kChunks / 32; ++e) {
                    const uint32_t at = st + L::kHalf + (lane + 32 * e) * 16;
                    const uint4 w = ptx::lds128(at);
                    ptx::sts128(at, make_uint4(finite2<F16>(w.x), finite2<F16>(w.y), finite2<F16>(w.z), finite2<F16>(w.w)));
                }
                __syncwarp();
            }
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t vb[4];
                const int row = ((lane >> 3) & 1) * 8 + (lane & 7), ch = 2 * d + (lane >> 4);
                ldm4t(vb, st + L::kHalf + row * HD * 2 + ((ch ^ (row & 7)) << 4));
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    mma16816<F16>(acc[a][2 * d], pa[a], vb[0], vb[1]);
                    mma16816<F16>(acc[a][2 * d + 1], pa[a], vb[2], vb[3]);
                }
            }
        }
        cp_wait<0>();
        // ---- merge the warps
#pragma unroll
        for (int y = 0; y < 2 * MT; ++y) {
            l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
            l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
            if ((lane & 3) == 0) {
                stat_m[warp * 16 * MT + 8 * y + (lane >> 2)] = m[y];
                stat_l[warp * 16 * MT + 8 * y + (lane >> 2)] = l[y];
            }
        }
        __syncthreads();                           // (every warp has left its K and V)
        float* const merge = reinterpret_cast<float*>(smem + L::kQ + L::kStats);
        {
            float* const mine = merge + warp * 16 * MT * HD;
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int d = 0; d < HD / 8; ++d) {
                    const int r = 16 * a + (lane >> 2), col = 8 * d + 2 * (lane & 3);
                    *reinterpret_cast<float2*>(mine + r * HD + (col ^ ((r & 3) << 3))) = make_float2(acc[a][d][0], acc[a][d][1]);
                    *reinterpret_cast<float2*>(mine + (r + 8) * HD + (col ^ ((r & 3) << 3))) = make_float2(acc[a][d][2], acc[a][d][3]);
                }
        }
        __syncthreads();
        // row r of the block, columns d .. d + 3, from its rows in `n` places (warps, or blocks of the cluster): the sum relative to
        // the largest of their maxima, which is left in `top`
        auto join = [&](int n, auto&& m_of, auto&& l_of, auto&& row_of, float& top, float& sum) {
            top = -INFINITY;
            for (int y = 0; y < n; ++y) top = fmaxf(top, m_of(y));
            const float b = top == -INFINITY ? 0.f : top;
            float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
            sum = 0.f;
#pragma unroll 4
            for (int y = 0; y < n; ++y) {
                const float w = ptx::ex2(m_of(y) - b);
                const float4 z = row_of(y);          // (zeros where no key of the row has been seen)
                sum = fmaf(w, l_of(y), sum);
                t.x = fmaf(w, z.x, t.x);
                t.y = fmaf(w, z.y, t.y);
                t.z = fmaf(w, z.z, t.z);
                t.w = fmaf(w, z.w, t.w);
            }
            return t;
        };
        // O and LSE of row rho, columns d .. d + 3, of which t is the sum; `none`: the row has seen no key (or all scores are -inf)
        auto store = [&](int rho, int d, float4 t, float top, float sum, bool none) {
            none = none || sum == 0.f;
            const int i = rho / p.G, h = hk * p.G + rho - i * p.G;
            const int64_t at = ((int64_t)s.b * p.H + h) * p.Nq + s.q0 + i;
            const float ll = none ? -INFINITY : (top + log2f(sum)) * kLn2, inv = none ? 0.f : 1.f / sum;
            if (none) t = make_float4(0.f, 0.f, 0.f, 0.f);
            t = make_float4(t.x * inv, t.y * inv, t.z * inv, t.w * inv);
            if (P.shares > 1 && !P.cluster) {
                if (!none) *reinterpret_cast<float4*>(P.part_o + (share * rows_all + at) * HD + d) = t;
                if (d == 0) P.part_lse[share * rows_all + at] = ll;
                return;
            }
            if (d == 0) lse[at] = ll;
            if (d >= p.D) return;
            const int64_t dst = s.b * p.o.b + (int64_t)(s.q0 + i) * p.o.n + h * p.o.h + d;
            uint2 y, low;
            pack_split<F16>(t.x, t.y, y.x, low.x);
            pack_split<F16>(t.z, t.w, y.y, low.y);
            *reinterpret_cast<uint2*>(o + dst) = y;
            if (o_low) *reinterpret_cast<uint2*>(o_low + dst) = low;
        };
        float* const block = merge + 4 * 16 * MT * HD;              // the block's rows, for the cluster
        for (int c = tid; c < 16 * MT * (HD / 4); c += kFewThreads) {
            const int r = c / (HD / 4), d = c % (HD / 4) * 4, rho = r0 + r;
            if (rho >= R) continue;
            float top, sum;
            const float4 t = join(4, [&](int y) { return stat_m[y * 16 * MT + r]; }, [&](int y) { return stat_l[y * 16 * MT + r]; },
                                  [&](int y) { return *reinterpret_cast<const float4*>(merge + (y * 16 * MT + r) * HD + (d ^ ((r & 3) << 3))); }, top, sum);
            if (P.cluster) {
                *reinterpret_cast<float4*>(block + r * HD + d) = t;
                if (d == 0) {
                    stat_m[4 * 16 * MT + r] = top;
                    stat_l[4 * 16 * MT + r] = sum;
                }
            } else {
                store(rho, d, t, top, sum, min(rho / p.G + s.off(), c1 - 1) < c0);
            }
        }
        if (P.cluster) {
            cluster_sync();
            // (16 MT HD / 4 items dealt out to the blocks)
            const uint32_t sm = ptx::smem_u32(stat_m + 4 * 16 * MT), sl = ptx::smem_u32(stat_l + 4 * 16 * MT), sb = ptx::smem_u32(block);
            for (int c = share + P.shares * tid; c < 16 * MT * (HD / 4); c += P.shares * kFewThreads) {
                const int r = c / (HD / 4), d = c % (HD / 4) * 4, rho = r0 + r;
                if (rho >= R) continue;
                float top, sum;
                const float4 t = join(P.shares, [&](int y) { return ld_cluster(of_rank(sm + r * 4, y)); }, [&](int y) { return ld_cluster(of_rank(sl + r * 4, y)); },
                                      [&](int y) { return ld_cluster4(of_rank(sb + (r * HD + d) * 4, y)); }, top, sum);
                store(rho, d, t, top, sum, rho / p.G + s.off() < 0);
            }
            cluster_sync();                        // (nobody leaves, or writes its rows anew, before all have read them)
        }
        __syncthreads();
    }
    if (p.cu_q != nullptr) {
        zero_outside(o, p.o, p.H, p.D, p.Nq, p.cu_q, p.S, blockIdx.x, gridDim.x);
        empty_lse_outside(lse, p.H, p.Nq, p.cu_q, p.S, blockIdx.x, gridDim.x);
    }
}

struct FewPlan {
    int mt, shares, steps, row_blocks;
    size_t part_o, part_lse, bytes;
};
// Shares of the keys, by an estimate of the time: a round of resident blocks (two to a multiprocessor) costs 1.5 us before its
// first and after its last step; a step takes 1 us, or what its bytes take of the bandwidth where all of them run; joining
// takes 1 us and round in a cluster, else 5 us and 0.05 for every share.
inline FewPlan plan_few(const CParams& c) {
    FewPlan f{};
    const int rows = (int)((int64_t)c.max_q * c.G < kFewRowsMost ? c.max_q * c.G : kFewRowsMost);
    f.mt = rows > 16 ? 2 : 1;
    f.row_blocks = ceil_div(rows, 16 * f.mt);
    const bool packed = c.cu_q != nullptr;
    const int longest = ceil_div(c.max_k, kFewKeys);
    const double heads = (double)c.Hkv * f.row_blocks, slots = 2.0 * host::sm_count();
    const double total = packed ? (double)c.Nk / kFewKeys + 0.5 * c.S : (double)longest * c.S;      // steps of a head
    double best = 1e30;
    // (a dozen of counts up to 16, then steps of an eighth: this runs on the host before every call)
    for (int n = 1, last = 0; n <= 128 && n <= longest; n += n < 16 ? 1 : n / 8) {
        const int per = ceil_div(longest, n);
        if (per == last) continue;
        last = per;
        const double blocks = heads * (packed ? (total / per < c.S ? c.S : total / per + 0.5 * c.S) : (double)ceil_div(longest, per) * c.S);
        double rounds = blocks / slots;
        rounds = rounds <= 1 ? 1 : rounds < 4 ? (double)(int)(rounds + 0.999) : rounds + 0.5;
        const double running = blocks < slots ? blocks : slots, bound = kFewKeys * c.D * 4.0 * running / 6.2e6;
        const double us = rounds * (1.5 + per * (bound > 1.0 ? bound : 1.0)) + (n > kFewCluster ? 5.0 + 0.05 * n : n > 1 ? 1.0 * rounds : 0.0);
        if (us < best) {
            best = us;
            f.shares = ceil_div(longest, per);
            f.steps = per;
        }
    }
    const size_t all = (size_t)c.B * c.H * c.Nq;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t x = at; at += (n + 255) / 256 * 256; return x; };
    const bool join = f.shares > kFewCluster;
    f.part_o = take(join ? (size_t)f.shares * all * tile_columns(c.D) * 4 : 0);
    f.part_lse = take(join ? (size_t)f.shares * all * 4 : 0);
    f.bytes = at;
    return f;
}

template <int HD, bool F16>
int launch_few(const CParams& c, const void* q, const void* k, const void* v, void* o, void* o_low, float* lse, uint8_t* ws, cudaStream_t st) {
    const FewPlan f = plan_few(c);
    const int64_t grid = (int64_t)c.S * c.Hkv * f.row_blocks * f.shares;
    if (grid > 0x7fffffff) return SA_ERR_UNSUPPORTED;
    FewParams P{};
    P.c = c;
    P.shares = f.shares;
    P.steps = f.steps;
    P.cluster = f.shares > 1 && f.shares <= kFewCluster;
    P.row_blocks = f.row_blocks;
    P.part_o = reinterpret_cast<float*>(ws + f.part_o);
    P.part_lse = reinterpret_cast<float*>(ws + f.part_lse);
    auto go = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        auto kern = causal_few_kernel<HD, F16, MT>;
        if (!allow_dynamic_smem((const void*)kern, FewLayout<HD, MT>::kBytes)) return SA_ERR_LAUNCH;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)f.shares;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3(kFewThreads);
        cfg.dynamicSmemBytes = FewLayout<HD, MT>::kBytes;
        cfg.stream = st;
        cfg.attrs = &attr;
        cfg.numAttrs = P.cluster ? 1 : 0;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (__nv_bfloat16*)o,
                                                 (__nv_bfloat16*)o_low, lse);
        host::count_launches(1);
        return e == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
    };
    const int rc = f.mt == 2 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 1>{});
    if (rc != SA_OK || f.shares == 1 || P.cluster) return rc;
    return launch_join<HD>(c, F16, f.shares, P.part_o, P.part_lse, o, o_low, lse, st);
}

}  // namespace causal
}  // namespace sa
