// Host services of the C entries, shared by the translation units (definitions in sa_api.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/simplicial_attn_b200.h"

namespace sa {
namespace host {

void count_launches(int n);
uint64_t wait_limit_ns();
int sm_count();           // of the current device, or a B200's where there is none
int cc_major();           // 0 where there is no device
// Tensor map over a 16-bit [B, rows, heads, D] tensor; a box is 64 elements of one row by `box_rows` rows, 128-byte swizzled.
bool make_map(CUtensorMap* map, const void* base, int B, int rows, int heads, int D, const sa_strides& st, int box_rows, bool f16);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool strides8(const sa_strides& s) { return s.b % 8 == 0 && s.n % 8 == 0 && s.h % 8 == 0; }

}  // namespace host
}  // namespace sa
