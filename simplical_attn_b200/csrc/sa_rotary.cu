// Rotary positions (sa_rotary): every pair (x, y) of the rotated part of a head turned by position * frequency.
//
// The kernel moves every element once and computes about three flops for it: HBM bandwidth bounds it, launch latency where
// there are few rows.  Nothing is tabulated beyond a block: an angle is formed from the position and the frequency, so any
// position works.  The product is taken and reduced to an eighth of a turn in 64 bits (in 32 a position of 10^6 would be off by
// 0.06 radians), sine and cosine of the remainder in 32.
//
// A thread turns two 16-byte vectors of each of up to four heads of a row.  Its loads are issued first; while they are under
// way the block makes the sines and cosines of its few rows in shared memory, once for all heads.
//
// Measured: 16384 rows of 32 + 2 heads of 128 in bf16 take 47.8 us (6.0 TB/s of their bytes; 84 us while every thread made its own
// sines and moved 16-bit elements one by one), a token of eight sequences 2.7 us in a graph.
#include <cuda_runtime.h>

#include "sa_common.cuh"
#include "sa_host.cuh"
#include "sa_ptx.cuh"

namespace sa {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kHeads = 4;            // heads a thread turns by the same angles
constexpr int kMaxTensors = 4;
constexpr int kMaxHalf = 1024;       // pairs of a head: bounds the table

struct Params {
    const void* in[kMaxTensors];
    void* out[kMaxTensors];
    sa_strides si[kMaxTensors], so[kMaxTensors];
    int heads[kMaxTensors];
    int blocks_end[kMaxTensors];     // head blocks of the tensors up to this one
    int tensors, N, D, rd;
    unsigned rows, head_blocks, groups, turned_groups;       // groups: of 2 V elements of a head
    unsigned table_rows;             // rows that a block's threads can be of
    const void* positions;
    const void* frequencies;
    int position_bits, frequency_bits;
    int64_t position_b, position_n, offset;
    float magnitude;
    int inverse;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};
template <> struct alignas(16) Vec<__half, 8> { uint32_t w[4]; };
template <> struct alignas(16) Vec<__nv_bfloat16, 8> { uint32_t w[4]; };
template <> struct alignas(8) Vec<__half, 4> { uint32_t w[2]; };
template <> struct alignas(8) Vec<__nv_bfloat16, 4> { uint32_t w[2]; };
template <> struct alignas(4) Vec<__half, 2> { uint32_t w[1]; };
template <> struct alignas(4) Vec<__nv_bfloat16, 2> { uint32_t w[1]; };

// cos and sin of a whole turn's fraction given in quarter turns: the nearest whole number of quarters is taken off in 64
// bits, so that the 32-bit remainder is at most an eighth of a turn and its rounding at most 2^-25 quarters.
__device__ __forceinline__ void cos_sin_quarters(double quarters, float& c, float& s) {
    const double n = rint(quarters);
    float sr, cr;
    sincospif(0.5f * (float)(quarters - n), &sr, &cr);
    const int k = (int)(n - 4.0 * floor(0.25 * n));        // n modulo 4
    c = (k & 1) ? sr : cr;
    s = (k & 1) ? cr : sr;
    if (k == 1 || k == 2) c = -c;
    if (k >= 2) s = -s;
}

__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
    const float u = x * c - y * s;
    y = y * c + x * s;
    x = u;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w) { return make_float2(ptx::El<std::is_same<T, __half>::value>::lo(w), ptx::El<std::is_same<T, __half>::value>::hi(w)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float2 v) { return ptx::El<std::is_same<T, __half>::value>::pack(v.x, v.y); }

// The pairs of two vectors, by the angles of theirs in the order of the elements.  16-bit elements are handled as the packed
// words that they are loaded as (one by one the compiler spent three times the instructions on moving halves about).
template <typename T, int V, bool INTERLEAVED>
__device__ __forceinline__ void turn_pairs(Vec<T, V>& a, Vec<T, V>& c, const float (&cs)[V], const float (&sn)[V]) {
    if constexpr (sizeof(T) == 2 && V >= 2) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            float2 x = unpack2<T>(a.w[e]), y = unpack2<T>(c.w[e]);
            if (INTERLEAVED) {
                turn(x.x, x.y, cs[e], sn[e]);
                turn(y.x, y.y, cs[V / 2 + e], sn[V / 2 + e]);
            } else {
                turn(x.x, y.x, cs[2 * e], sn[2 * e]);
                turn(x.y, y.y, cs[2 * e + 1], sn[2 * e + 1]);
            }
            a.w[e] = pack2<T>(x);
            c.w[e] = pack2<T>(y);
        }
    } else {
        float x[2 * V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[e] = to_f<T>(a.e[e]);
            x[V + e] = to_f<T>(c.e[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) turn(x[INTERLEAVED ? 2 * e : e], x[INTERLEAVED ? 2 * e + 1 : V + e], cs[e], sn[e]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            a.e[e] = from_f<T>(x[e]);
            c.e[e] = from_f<T>(x[V + e]);
        }
    }
}

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(const __grid_constant__ Params p) {
    extern __shared__ float4 table4[];
    const int half = p.rd / 2, pitch = (half + 3) & ~3;            // angles of a row
    float* const cosines = reinterpret_cast<float*>(table4);
    float* const sines = cosines + p.table_rows * pitch;
    const unsigned per_row = p.groups * p.head_blocks;
    const unsigned row0 = blockIdx.x * kThreads / per_row, nrows = min((blockIdx.x * kThreads + kThreads - 1) / per_row + 1, p.rows) - row0;
    unsigned idx = blockIdx.x * kThreads + threadIdx.x;
    const unsigned g = idx % p.groups;
    idx /= p.groups;
    const unsigned hb = idx % p.head_blocks, row = min(idx / p.head_blocks, p.rows - 1);
    const bool live = idx / p.head_blocks < p.rows;
    const unsigned b = row / (unsigned)p.N, n = row - b * (unsigned)p.N;

    int t = 0, first_block = 0;
#pragma unroll
    for (int x = 0; x < kMaxTensors - 1; ++x)
        if (x + 1 < p.tensors && (int)hb >= p.blocks_end[x]) {
            t = x + 1;
            first_block = p.blocks_end[x];
        }
    // (selected by comparisons: an index that is not a constant would copy the parameters to local memory)
    const void* in = p.in[0];
    void* out = p.out[0];
    sa_strides si = p.si[0], so = p.so[0];
    int heads = p.heads[0];
#pragma unroll
    for (int x = 1; x < kMaxTensors; ++x)
        if (t == x) {
            in = p.in[x];
            out = p.out[x];
            si = p.si[x];
            so = p.so[x];
            heads = p.heads[x];
        }
    const int h0 = ((int)hb - first_block) * kHeads, nh = live ? min(kHeads, heads - h0) : 0;

    // the two vectors of this group within a head, half of the turned (or of the other) elements apart, so that neighbouring
    // threads read neighbouring vectors: the partners of half-split pairs, or V / 2 interleaved pairs each
    const bool turned = g < p.turned_groups;
    int oa, ob;
    if (!turned) {
        oa = p.rd + (int)(g - p.turned_groups) * V;
        ob = oa + (int)(p.groups - p.turned_groups) * V;
    } else if (INTERLEAVED && V == 1) {
        oa = 2 * (int)g;
        ob = oa + 1;
    } else {
        oa = (int)g * V;
        ob = p.rd / 2 + oa;
    }
    const bool have_b = ob < p.D;
    const T* src = (const T*)in + (int64_t)b * si.b + (int64_t)n * si.n + (int64_t)h0 * si.h;
    T* dst = (T*)out + (int64_t)b * so.b + (int64_t)n * so.n + (int64_t)h0 * so.h;
    const bool same = !turned && src == dst;                       // in place: nothing to copy

    using W = Vec<T, V>;
    W a[kHeads], c[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
        if (h < nh) {
            a[h] = *reinterpret_cast<const W*>(src + h * si.h + oa);
            if (have_b) c[h] = *reinterpret_cast<const W*>(src + h * si.h + ob);
        }
    for (unsigned z = threadIdx.x; z < nrows * half; z += kThreads) {
        const unsigned r = z / half, i = z - r * half, yb = (row0 + r) / (unsigned)p.N, yn = row0 + r - yb * (unsigned)p.N;
        int64_t at = p.offset;
        if (p.positions == nullptr) at += yn;
        else {
            const int64_t y = (int64_t)yb * p.position_b + (int64_t)yn * p.position_n;
            at += p.position_bits == 64 ? ((const int64_t*)p.positions)[y] : (int64_t)((const int32_t*)p.positions)[y];
        }
        const double f = p.frequency_bits == 64 ? ((const double*)p.frequencies)[i] : (double)((const float*)p.frequencies)[i];
        float cs, sn;
        cos_sin_quarters((double)at * 0.63661977236758134308 * f, cs, sn);      // 2 / pi
        cosines[r * pitch + i] = cs * p.magnitude;
        sines[r * pitch + i] = sn * (p.inverse ? -p.magnitude : p.magnitude);
    }
    __syncthreads();
    if (same) return;
    if (turned) {
        float cs[V], sn[V];
        auto angles = [&](const float* table, float (&v)[V]) {
            table += (row - row0) * pitch;
            if constexpr (V >= 4 && !INTERLEAVED) {
#pragma unroll
                for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(&v[e]) = *reinterpret_cast<const float4*>(table + oa + e);
            } else if constexpr (V == 8) {
                *reinterpret_cast<float4*>(&v[0]) = *reinterpret_cast<const float4*>(table + oa / 2);
                *reinterpret_cast<float4*>(&v[4]) = *reinterpret_cast<const float4*>(table + ob / 2);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    v[e] = table[!INTERLEAVED ? oa + e : V == 1 ? oa / 2 : (e < V / 2 ? oa : ob) / 2 + e % (V / 2 ? V / 2 : 1)];
            }
        };
        angles(cosines, cs);
        angles(sines, sn);
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
            if (h < nh) turn_pairs<T, V, INTERLEAVED>(a[h], c[h], cs, sn);
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
        if (h < nh) {
            *reinterpret_cast<W*>(dst + h * so.h + oa) = a[h];
            if (have_b) *reinterpret_cast<W*>(dst + h * so.h + ob) = c[h];
        }
}

template <typename T, int V>
int launch_v(Params& p, bool interleaved, cudaStream_t st) {
    p.turned_groups = (unsigned)(p.rd / (2 * V));
    p.groups = p.turned_groups + (unsigned)((p.D - p.rd + 2 * V - 1) / (2 * V));
    const uint64_t threads = (uint64_t)p.rows * p.head_blocks * p.groups;
    if (threads > 0x7fffffffull - kThreads) return SA_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)((threads + kThreads - 1) / kThreads), pitch = (unsigned)(p.rd / 2 + 3) & ~3u;
    // (at most (256 / groups + 2) (V groups + 4) angles: 32 KB)
    p.table_rows = kThreads / (p.head_blocks * p.groups) + 2;
    if (p.table_rows > p.rows) p.table_rows = p.rows;
    const size_t smem = 2 * sizeof(float) * p.table_rows * pitch;
    if (p.rd / 2 > kMaxHalf || smem > 48 * 1024) return SA_ERR_UNSUPPORTED;
    if (interleaved) rotary_kernel<T, V, true><<<grid, kThreads, smem, st>>>(p);
    else rotary_kernel<T, V, false><<<grid, kThreads, smem, st>>>(p);
    host::count_launches(1);
    return cudaGetLastError() == cudaSuccess ? SA_OK : SA_ERR_LAUNCH;
}

// The widest vectors (up to 16 bytes) that every address of the call allows.
template <typename T>
int launch_t(Params& p, bool interleaved, cudaStream_t st) {
    auto fits = [&](int v) {
        if (p.rd % (2 * v) != 0 || p.D % v != 0) return false;
        for (int t = 0; t < p.tensors; ++t) {
            if (reinterpret_cast<uintptr_t>(p.in[t]) % (v * sizeof(T)) != 0 || reinterpret_cast<uintptr_t>(p.out[t]) % (v * sizeof(T)) != 0) return false;
            for (const sa_strides* s : {&p.si[t], &p.so[t]})
                if (s->b % v != 0 || s->n % v != 0 || s->h % v != 0) return false;
        }
        return true;
    };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch_v<T, 8>(p, interleaved, st);
    if (fits(4)) return launch_v<T, 4>(p, interleaved, st);
    if (fits(2)) return launch_v<T, 2>(p, interleaved, st);
    return launch_v<T, 1>(p, interleaved, st);
}

}  // namespace rotary
}  // namespace sa

extern "C" int sa_rotary(const sa_rotary_params* p, const void* const* in, void* const* out, const void* positions,
                         const void* frequencies, void* stream) {
    using namespace sa::rotary;
    if (!p || !in || !out || !frequencies) return SA_ERR_NULL_POINTER;
    if (p->tensors < 1 || p->tensors > kMaxTensors || p->B < 1 || p->N < 1 || p->D < 1) return SA_ERR_BAD_SHAPE;
    if (p->rotary_dim < 2 || p->rotary_dim > p->D || p->rotary_dim % 2 != 0) return SA_ERR_BAD_SHAPE;
    if (p->dtype < SA_BF16 || p->dtype > SA_F32) return SA_ERR_UNSUPPORTED;
    if (p->frequency_bits != 32 && p->frequency_bits != 64) return SA_ERR_UNSUPPORTED;
    if (positions && p->position_bits != 32 && p->position_bits != 64) return SA_ERR_UNSUPPORTED;
    if ((int64_t)p->B * p->N > 0x7fffffffll) return SA_ERR_UNSUPPORTED;
    Params k{};
    int blocks = 0;
    for (int t = 0; t < p->tensors; ++t) {
        if (!in[t] || !out[t]) return SA_ERR_NULL_POINTER;
        if (p->heads[t] < 1) return SA_ERR_BAD_SHAPE;
        k.in[t] = in[t];
        k.out[t] = out[t];
        k.si[t] = p->in[t];
        k.so[t] = p->out[t];
        for (sa_strides* x : {&k.si[t], &k.so[t]}) {       // the stride of an extent of one is never used
            if (p->B == 1) x->b = 0;
            if (p->N == 1) x->n = 0;
            if (p->heads[t] == 1) x->h = 0;
        }
        k.heads[t] = p->heads[t];
        blocks += (p->heads[t] + kHeads - 1) / kHeads;
        k.blocks_end[t] = blocks;
    }
    k.tensors = p->tensors;
    k.N = p->N;
    k.D = p->D;
    k.rd = p->rotary_dim;
    k.rows = (unsigned)(p->B * p->N);
    k.head_blocks = (unsigned)blocks;
    k.positions = positions;
    k.frequencies = frequencies;
    k.position_bits = p->position_bits;
    k.frequency_bits = p->frequency_bits;
    k.position_b = p->position_b;
    k.position_n = p->position_n;
    k.offset = p->offset;
    k.magnitude = p->magnitude;
    k.inverse = p->inverse != 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool il = p->interleaved != 0;
    if (p->dtype == SA_BF16) return launch_t<__nv_bfloat16>(k, il, st);
    if (p->dtype == SA_F16) return launch_t<__half>(k, il, st);
    return launch_t<float>(k, il, st);
}
