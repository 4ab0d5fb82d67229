// C entries of causal attention: argument validation, kernel selection and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "sa_causal.cuh"
#include "sa_causal_bwd.cuh"
#include "sa_causal_few.cuh"
#include "sa_causal_fwd.cuh"
#include "sa_causal_general.cuh"

namespace sa {
namespace causal {
namespace {

int validate(const sa_causal_params* p) {
    if (!p) return SA_ERR_NULL_POINTER;
    if (p->B < 1 || p->Nq < 1 || p->Nk < 1 || p->H < 1 || p->Hkv < 1 || p->D < 1 || p->H % p->Hkv != 0) return SA_ERR_BAD_SHAPE;
    if (p->sequences < 0 || p->max_q < 0 || p->max_k < 0 || (p->sequences > 0 && p->B != 1)) return SA_ERR_BAD_SHAPE;
    if (p->dtype < SA_BF16 || p->dtype > SA_F32 || p->D > 256) return SA_ERR_UNSUPPORTED;
    if (p->algo < SA_ALGO_AUTO || p->algo > SA_ALGO_TCGEN05) return SA_ERR_UNSUPPORTED;
    if ((int64_t)p->B * p->H * p->Nq > 0x7fffffff || (int64_t)p->B * p->Hkv * p->Nk > 0x7fffffff) return SA_ERR_UNSUPPORTED;
    if (p->Nq > (1 << 30) || p->Nk > (1 << 30) || (int64_t)p->H * (p->sequences > 0 ? p->sequences : p->B) > (1 << 30)) return SA_ERR_UNSUPPORTED;
    return SA_OK;
}

CParams make_params(const sa_causal_params* p, const int32_t* cu_q, const int32_t* cu_k) {
    CParams c{};
    c.B = p->B; c.Nq = p->Nq; c.Nk = p->Nk; c.H = p->H; c.Hkv = p->Hkv; c.D = p->D; c.G = p->H / p->Hkv;
    c.S = p->sequences > 0 ? p->sequences : p->B;
    c.max_q = p->sequences > 0 && p->max_q > 0 && p->max_q < p->Nq ? p->max_q : p->Nq;
    c.max_k = p->sequences > 0 && p->max_k > 0 && p->max_k < p->Nk ? p->max_k : p->Nk;
    c.cu_q = cu_q; c.cu_k = cu_k;
    c.scale = p->scale;
    c.q = p->q; c.k = p->k; c.v = p->v; c.o = p->o; c.d_o = p->d_o; c.dq = p->dq; c.dk = p->dk; c.dv = p->dv;
    // the stride of an extent of one is never used
    auto fix = [](sa_strides& s, int b, int n, int h) {
        if (b == 1) s.b = 0;
        if (n == 1) s.n = 0;
        if (h == 1) s.h = 0;
    };
    for (sa_strides* s : {&c.q, &c.o, &c.d_o, &c.dq}) fix(*s, c.B, c.Nq, c.H);
    for (sa_strides* s : {&c.k, &c.v, &c.dk, &c.dv}) fix(*s, c.B, c.Nk, c.Hkv);
    return c;
}

// Whether the tensor-core kernels cover the problem (pointers and what a tensor map can hold are looked at in the call).
bool tc_ok(const sa_causal_params* p, bool backward) {
    if (p->dtype == SA_F32 || p->D > 128 || p->D % 8 != 0) return false;
    if (!(p->scale > 0.f)) return false;            // the row maximum is taken before scaling
    const CParams c = make_params(p, nullptr, nullptr);
    for (const sa_strides* s : {&c.q, &c.k, &c.v, &c.o})
        if (!host::strides8(*s)) return false;
    if (backward)
        for (const sa_strides* s : {&c.d_o, &c.dq, &c.dk, &c.dv})
            if (!host::strides8(*s)) return false;
    return true;
}

int resolve(const sa_causal_params* p, bool backward) {
    const bool ok = p->algo != SA_ALGO_GENERAL && tc_ok(p, backward);
    if (p->algo == SA_ALGO_TCGEN05) return ok ? SA_ALGO_TCGEN05 : -SA_ERR_UNSUPPORTED;
    if (!ok) return SA_ALGO_GENERAL;
    const CParams c = make_params(p, nullptr, nullptr);
    return !backward && (int64_t)c.max_q * c.G <= kFewRowsMost ? (int)SA_CAUSAL_FEW_ROWS : (int)SA_ALGO_TCGEN05;
}

// (a plan only asks whether there are starts)
const int32_t* const kSomeStarts = reinterpret_cast<const int32_t*>(64);
CParams planned(const sa_causal_params* p) {
    const int32_t* cu = p->sequences > 0 ? kSomeStarts : nullptr;
    return make_params(p, cu, cu);
}

// f(columns of a tile, element type) of the tensor-core kernels
template <typename F>
int dispatch_tc(const sa_causal_params* p, F&& f) {
    auto by_type = [&](auto d) { return p->dtype == SA_F16 ? f(d, std::true_type{}) : f(d, std::false_type{}); };
    return tile_columns(p->D) == 128 ? by_type(std::integral_constant<int, 128>{}) : by_type(std::integral_constant<int, 64>{});
}

bool workspace_ok(const void* ws, size_t bytes, size_t need) {
    if (need == 0) return true;
    return ws != nullptr && bytes >= need && (reinterpret_cast<uintptr_t>(ws) & 255u) == 0;
}

}  // namespace
}  // namespace causal
}  // namespace sa

extern "C" {

size_t sa_causal_forward_workspace_size(const sa_causal_params* p) {
    using namespace sa::causal;
    if (validate(p) != SA_OK) return 0;
    const int algo = resolve(p, false);
    if (algo < 0) return 0;
    // (a call whose pointers or strides turn out not to suit the tensor cores takes the general kernels)
    const CParams c = planned(p);
    const size_t general = plan_general(c, false).bytes, own = algo == SA_ALGO_TCGEN05 ? plan_fwd(c).bytes : algo == SA_CAUSAL_FEW_ROWS ? plan_few(c).bytes : 0;
    return general > own ? general : own;
}

size_t sa_causal_backward_workspace_size(const sa_causal_params* p) {
    using namespace sa::causal;
    if (validate(p) != SA_OK) return 0;
    const int algo = resolve(p, true);
    if (algo < 0) return 0;
    const CParams c = planned(p);
    const size_t general = plan_general(c, true).bytes, own = algo == SA_ALGO_TCGEN05 ? plan_bwd(c, p->dtype == SA_F16).bytes : 0;
    return general > own ? general : own;
}

int sa_causal_resolve(const sa_causal_params* p, int backward) {
    using namespace sa::causal;
    const int rc = validate(p);
    return rc != SA_OK ? -rc : resolve(p, backward != 0);
}

int sa_causal_forward(const sa_causal_params* p, const void* q, const void* k, const void* v, void* o, void* o_low, float* lse,
                      const int32_t* cu_q, const int32_t* cu_k, void* workspace, size_t workspace_bytes, void* status, void* stream) try {
    using namespace sa::causal;
    int rc = validate(p);
    if (rc != SA_OK) return rc;
    if (!q || !k || !v || !o || !lse || !status || (p->sequences > 0 && (!cu_q || !cu_k))) return SA_ERR_NULL_POINTER;
    if (!workspace_ok(workspace, workspace_bytes, sa_causal_forward_workspace_size(p)) || !sa::host::aligned16(status)) return SA_ERR_WORKSPACE;
    const int algo = resolve(p, false);
    if (algo < 0) return -algo;
    const CParams c = make_params(p, p->sequences > 0 ? cu_q : nullptr, p->sequences > 0 ? cu_k : nullptr);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (algo != SA_ALGO_GENERAL) {
        if (sa::host::cc_major() != 10) return SA_ERR_NOT_SM100;
        rc = SA_ERR_BAD_STRIDE;
        if (sa::host::aligned16(q) && sa::host::aligned16(k) && sa::host::aligned16(v) && sa::host::aligned16(o) && sa::host::aligned16(o_low))
            rc = dispatch_tc(p, [&](auto d, auto f16) {
                if (algo == SA_CAUSAL_FEW_ROWS)
                    return launch_few<decltype(d)::value, decltype(f16)::value>(c, q, k, v, o, o_low, lse, static_cast<uint8_t*>(workspace), st);
                return launch_fwd_tc<decltype(d)::value, decltype(f16)::value>(c, q, k, v, o, o_low, lse, static_cast<uint8_t*>(workspace),
                                                                             static_cast<sa::DeviceStatus*>(status), st);
            });
        // (BAD_STRIDE: nothing has been launched)
        if (rc != SA_ERR_BAD_STRIDE || p->algo == SA_ALGO_TCGEN05) return rc;
    }
    return dispatch_general(p->dtype, p->D, [&](auto t, auto d) { return launch_general_fwd_d<decltype(t), decltype(d)::value>(c, q, k, v, o, o_low, lse, static_cast<uint8_t*>(workspace), st); });
} catch (...) {      // (no C++ exception leaves a C entry: out of host memory)
    return SA_ERR_LAUNCH;
}

int sa_causal_backward(const sa_causal_params* p, const void* q, const void* k, const void* v, const void* o, const void* o_low, const float* lse,
                       const void* d_o, void* dq, void* dk, void* dv, const int32_t* cu_q, const int32_t* cu_k, void* workspace, size_t workspace_bytes, void* status,
                       void* stream) try {
    using namespace sa::causal;
    int rc = validate(p);
    if (rc != SA_OK) return rc;
    if (!q || !k || !v || !o || !lse || !d_o || !status || (p->sequences > 0 && (!cu_q || !cu_k))) return SA_ERR_NULL_POINTER;
    if (!workspace_ok(workspace, workspace_bytes, sa_causal_backward_workspace_size(p)) || !sa::host::aligned16(status)) return SA_ERR_WORKSPACE;
    if (!dq && !dk && !dv) return SA_OK;
    const int algo = resolve(p, true);
    if (algo < 0) return -algo;
    const CParams c = make_params(p, p->sequences > 0 ? cu_q : nullptr, p->sequences > 0 ? cu_k : nullptr);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (algo == SA_ALGO_TCGEN05) {
        if (sa::host::cc_major() != 10) return SA_ERR_NOT_SM100;
        rc = SA_ERR_BAD_STRIDE;
        bool aligned = true;
        for (const void* x : {q, k, v, o, o_low, d_o, (const void*)dq, (const void*)dk, (const void*)dv}) aligned = aligned && sa::host::aligned16(x);
        if (aligned)
            rc = dispatch_tc(p, [&](auto d, auto f16) {
                return launch_bwd_tc<decltype(d)::value, decltype(f16)::value>(c, q, k, v, o, o_low, lse, d_o, dq, dk, dv, static_cast<uint8_t*>(workspace),
                                                                             static_cast<sa::DeviceStatus*>(status), st);
            });
        if (rc != SA_ERR_BAD_STRIDE || p->algo == SA_ALGO_TCGEN05) return rc;
    }
    return dispatch_general(p->dtype, p->D, [&](auto t, auto d) {
        return launch_general_bwd_d<decltype(t), decltype(d)::value>(c, q, k, v, o, o_low, lse, d_o, dq, dk, dv, static_cast<uint8_t*>(workspace), st);
    });
} catch (...) {
    return SA_ERR_LAUNCH;
}

}  // extern "C"
