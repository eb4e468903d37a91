// The paged K/V cache of grouped heads (MI355X, gfx950): new rows written into their
// slots, and rows of slots read back in bf16.
//
// A slot is block * page + row. A bf16 cache holds the rows as they are. An fp8 cache
// holds, for each row (one token and kv head, D dims), e4m3fn codes and one fp32
// scale: scale = max(amax / 448, 2^-126) with amax over the row's finite values,
// code = e4m3fn(x / scale), nearest even; a value that is not finite becomes a NaN
// code. Reading gives bf16(code * scale).
//
// HBM bound: 2 bytes of a value on one side, 1 (and 4 / D of the scale) or 2 on the
// other. A thread holds 16 bytes of the cached row (16 or 8 values) of K and of V, so
// four or two wide loads are in flight before it waits; a row's D / 16 or D / 8
// threads lie side by side in one wave, which reduces amax without LDS. Written rows go
// past the caches: 16384 tokens of 8 heads of 128 dims in fp8 17.9 us, 5.5 TB/s (20.2
// through them). Rows read, and their copies, go through them: 8192 such tokens 11.5
// us (13.1 to 15 with either past them), 4.3 TB/s with the launch.
#include <limits.h>

#include "gqa_common.hpp"

namespace mm {
namespace gqa {

constexpr int kThreads = 256;

struct RowsArgs {
  const char *k, *v;       // [N, Hkv, D] bf16 by strides (read) or the rows to fill
  long long k_s[2], v_s[2];  // token, head; elements
  Cache kc, vc;
  const int* slots;
  long long n;
  int heads, page_shift;
  long long num_slots;
};

__device__ __forceinline__ long long row_at(const Cache& c, int slot, int shift, int head) {
  return (slot >> shift) * c.block_s + head * c.head_s + (slot & ((1 << shift) - 1)) * c.row_s;
}
__device__ __forceinline__ long long scale_at(const Cache& c, int slot, int shift, int head) {
  return (slot >> shift) * c.sblock_s + head * c.shead_s + (slot & ((1 << shift) - 1));
}

// The largest finite magnitude of a pair, as fp32 bits.
__device__ __forceinline__ uint32_t finite_max(uint32_t m, uint32_t pair) {
  const uint32_t lo = (pair << 16) & 0x7FFF0000u, hi = pair & 0x7FFF0000u;
  m = max(m, lo < 0x7F800000u ? lo : 0u);
  return max(m, hi < 0x7F800000u ? hi : 0u);
}

// 16 bf16 values of a row -> their codes, and the row's scale. LANES threads, side by
// side, hold the row.
template <int LANES>
__device__ __forceinline__ u32x4 quantize(const u32x4& x0, const u32x4& x1, float& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = finite_max(finite_max(m, x0[i]), x1[i]);
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  const float s = fmaxf(__builtin_bit_cast(float, m) / kFp8Max, kMinScale);
  const float r = 1.f / s;
  // x / s correctly rounded from the rounded reciprocal by one step on the exact
  // remainder (Markstein): 3 instructions instead of a division's 10, which would be
  // half of the kernel's time. An infinity's remainder is NaN, and so its code; a
  // zero's is +0, which would take the sign of -0.
  const auto div = [&](float x) {
    const float q = x * r;
    return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, s, x), r, q), x);
  };
  u32x4 out;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t p0 = (w < 2 ? x0 : x1)[(w & 1) * 2], p1 = (w < 2 ? x0 : x1)[(w & 1) * 2 + 1];
    s16x2 c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, div(bf16_lo(p0)), div(bf16_hi(p0)), 1.0f, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, div(bf16_lo(p1)), div(bf16_hi(p1)), 1.0f, true);
    out[w] = __builtin_bit_cast(uint32_t, c);
  }
  scale = s;
  return out;
}

template <int D, bool FP8>
__global__ __launch_bounds__(kThreads) void gqa_write_kernel(const RowsArgs a) {
  constexpr int kLanes = FP8 ? D / 16 : D / 8;  // threads of a row
  const long long item = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = item / kLanes;
  const int c = (int)(item % kLanes);
  if (row >= a.n * a.heads) return;  // whole rows: a wave's rows end together
  const long long tok = row / a.heads;
  const int head = (int)(row - tok * a.heads);
  const char* kp = a.k + 2 * (tok * a.k_s[0] + head * a.k_s[1]) + c * (FP8 ? 32 : 16);
  const char* vp = a.v + 2 * (tok * a.v_s[0] + head * a.v_s[1]) + c * (FP8 ? 32 : 16);
  const u32x4 k0 = *reinterpret_cast<const u32x4*>(kp), v0 = *reinterpret_cast<const u32x4*>(vp);
  u32x4 k1{}, v1{};
  if constexpr (FP8) {
    k1 = *reinterpret_cast<const u32x4*>(kp + 16);
    v1 = *reinterpret_cast<const u32x4*>(vp + 16);
  }
  const int slot = a.slots[tok];
  // The rows are loaded before the slot is tested, not a round trip behind it.
  asm volatile("" ::"v"(k0), "v"(v0), "v"(k1), "v"(v1));
  const bool live = slot >= 0 && slot < a.num_slots;  // else a padding token: nothing is written
  u32x4 ko = k0, vo = v0;
  float ks = 0.f, vs = 0.f;
  if constexpr (FP8) {
    ko = quantize<kLanes>(k0, k1, ks);
    vo = quantize<kLanes>(v0, v1, vs);
  }
  if (!live) return;
  constexpr int kElem = FP8 ? 1 : 2;
  __builtin_nontemporal_store(ko, reinterpret_cast<u32x4*>(a.kc.base + row_at(a.kc, slot, a.page_shift, head) * kElem + 16 * c));
  __builtin_nontemporal_store(vo, reinterpret_cast<u32x4*>(a.vc.base + row_at(a.vc, slot, a.page_shift, head) * kElem + 16 * c));
  if (FP8 && c == 0) {
    a.kc.scale[scale_at(a.kc, slot, a.page_shift, head)] = ks;
    a.vc.scale[scale_at(a.vc, slot, a.page_shift, head)] = vs;
  }
}

// 16 codes -> 16 bf16 values of code * scale.
__device__ __forceinline__ void dequantize(const u32x4& x, float s, u32x4& y0, u32x4& y1) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const u32x2 p = fp8x4_to_bf16(x[w]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      (w < 2 ? y0 : y1)[(w & 1) * 2 + h] = pack2_bf16_canon<kRTNE>(bf16_lo(p[h]) * s, bf16_hi(p[h]) * s);
  }
}

template <int D, bool FP8>
__global__ __launch_bounds__(kThreads) void gqa_read_kernel(const RowsArgs a) {
  constexpr int kLanes = FP8 ? D / 16 : D / 8;
  constexpr int kElem = FP8 ? 1 : 2;
  const long long item = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = item / kLanes;
  const int c = (int)(item % kLanes);
  if (row >= a.n * a.heads) return;
  const long long tok = row / a.heads;
  const int head = (int)(row - tok * a.heads);
  const int slot = a.slots[tok];
  u32x4 k0{}, k1{}, v0{}, v1{};  // a padding token's rows are zeros
  if (slot >= 0 && slot < a.num_slots) {
    k0 = *reinterpret_cast<const u32x4*>(a.kc.base + row_at(a.kc, slot, a.page_shift, head) * kElem + 16 * c);
    v0 = *reinterpret_cast<const u32x4*>(a.vc.base + row_at(a.vc, slot, a.page_shift, head) * kElem + 16 * c);
    if constexpr (FP8) {
      const float ks = a.kc.scale[scale_at(a.kc, slot, a.page_shift, head)];
      const float vs = a.vc.scale[scale_at(a.vc, slot, a.page_shift, head)];
      const u32x4 x = k0, y = v0;
      dequantize(x, ks, k0, k1);
      dequantize(y, vs, v0, v1);
    }
  }
  char* kp = const_cast<char*>(a.k) + 2 * (tok * a.k_s[0] + head * a.k_s[1]) + c * (FP8 ? 32 : 16);
  char* vp = const_cast<char*>(a.v) + 2 * (tok * a.v_s[0] + head * a.v_s[1]) + c * (FP8 ? 32 : 16);
  *reinterpret_cast<u32x4*>(kp) = k0;
  *reinterpret_cast<u32x4*>(vp) = v0;
  if constexpr (FP8) {
    *reinterpret_cast<u32x4*>(kp + 16) = k1;
    *reinterpret_cast<u32x4*>(vp + 16) = v1;
  }
}

int launch_rows(bool write, const void* k, const void* v, const void* k_cache, const void* v_cache,
                const void* k_scale, const void* v_scale, const void* slots, long long n, int heads, int D,
                int num_blocks, int page, const long long* st, void* stream) {
  if (D != 64 && D != 128 && D != 256) return -2;
  if (heads < 1) return -3;
  if (n < 0) return -4;
  if (page < 16 || (page & (page - 1)) != 0) return -5;
  if (num_blocks < 0 || (long long)num_blocks * page > (1LL << 31)) return -11;
  if (n == 0) return 0;
  if (!k || !v || !slots || !st || !k_scale != !v_scale) return -6;
  if (num_blocks > 0 && (!k_cache || !v_cache)) return -6;
  RowsArgs a{};
  a.k = (const char*)k;
  a.v = (const char*)v;
  for (int i = 0; i < 2; ++i) {
    a.k_s[i] = st[i];
    a.v_s[i] = st[2 + i];
  }
  a.kc = make_cache(k_cache, k_scale, st + 4);
  a.vc = make_cache(v_cache, v_scale, st + 9);
  a.slots = (const int*)slots;
  a.n = n;
  a.heads = heads;
  a.page_shift = __builtin_ctz(page);
  a.num_slots = (long long)num_blocks * page;
  const bool fp8 = k_scale != nullptr;
  const int lanes = fp8 ? D / 16 : D / 8;
  const long long grid = (n * heads * lanes + kThreads - 1) / kThreads;
  if (grid > UINT_MAX / kThreads) return -8;
  void (*kern)(RowsArgs);
#define MM_PICK(K)                                                     \
  (fp8 ? (D == 64 ? K<64, true> : D == 128 ? K<128, true> : K<256, true>) \
       : (D == 64 ? K<64, false> : D == 128 ? K<128, false> : K<256, false>))
  kern = write ? MM_PICK(gqa_write_kernel) : MM_PICK(gqa_read_kernel);
#undef MM_PICK
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

}  // namespace gqa
}  // namespace mm

extern "C" {

int launch_gqa_kv_write(const void* k, const void* v, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                        const void* slots, long long n_tokens, int Hkv, int head_dim, int num_blocks, int page,
                        const long long* strides, void* stream) {
  return mm::gqa::launch_rows(true, k, v, k_cache, v_cache, k_scale, v_scale, slots, n_tokens, Hkv, head_dim,
                              num_blocks, page, strides, stream);
}

int launch_gqa_kv_read(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                       const void* slots, void* k, void* v, long long n_tokens, int Hkv, int head_dim, int num_blocks,
                       int page, const long long* strides, void* stream) {
  return mm::gqa::launch_rows(false, k, v, k_cache, v_cache, k_scale, v_scale, slots, n_tokens, Hkv, head_dim,
                              num_blocks, page, strides, stream);
}

}  // extern "C"
