// Shared by the kernels over a paged K/V cache of grouped heads (gfx950): how a
// cache lies in memory, and its fp8 conversions.
#pragma once

#include "mm_common.hpp"

namespace mm {
namespace gqa {

// One of the two caches: element (block, head, row, d) lies at
// base[block * block_s + head * head_s + row * row_s + d] (strides in elements),
// the scale of a row (fp8) at scale[block * sblock_s + head * shead_s + row].
struct Cache {
  char* base;
  float* scale;
  long long block_s, head_s, row_s, sblock_s, shead_s;
};

// As the C ABI passes it: {block, head, row, scale block, scale head}.
inline Cache make_cache(const void* base, const void* scale, const long long* st) {
  return Cache{(char*)base, (float*)scale, st[0], st[1], st[2], st[3], st[4]};
}

constexpr float kFp8Max = 448.f;               // the largest e4m3fn value
constexpr float kMinScale = 1.17549435e-38f;   // 2^-126: x / scale stays finite for every bf16 row

typedef short s16x2 __attribute__((ext_vector_type(2)));

// Four e4m3fn codes -> four bf16 values (exact: e4m3fn is a subset of bf16), in order.
__device__ __forceinline__ u32x2 fp8x4_to_bf16(uint32_t codes) {
  u32x2 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true));
  return r;
}

__device__ __forceinline__ float bf16_lo(uint32_t pair) { return __builtin_bit_cast(float, pair << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t pair) { return __builtin_bit_cast(float, pair & 0xFFFF0000u); }

}  // namespace gqa
}  // namespace mm
