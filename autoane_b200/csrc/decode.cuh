// decode.cuh — shared by the decoding operators (kv_cache.cu, attn_prefix*.cu):
// the checked form of a b2p_kv_cache, and the widening of 8-bit codes to 16 bit.
#pragma once
#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "engine.cuh"
#include "mma.cuh"

namespace b2p {

constexpr int kKvHeadDim = 64;

struct KvView {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int n_pages, page_shift, kv_heads, kind;
  // Index of token `off` of page `page`, KV head h, in the scale arrays (64 codes each).
  __device__ __forceinline__ long long vec(int page, int h, int off) const {
    return (((long long)page * kv_heads + h) << page_shift) + off;
  }
};

// Checks a caller's cache (host side) and gives the kernels' form of it.
int kv_view(const b2p_kv_cache* c, int dtype, KvView* out);

// Four int8 codes (bytes of w) as 16-bit pairs (codes 0, 1) and (2, 3), exactly. fp16: 0x6400 | u is
// 1024 + u, so the code with its sign bit flipped (u = code + 128) less 1152 is the code. bf16 has
// 7 fraction bits: 0x4300 | low 7 bits is 128 + low, and 0x4300 | the sign bit is 128 or 256.
template <typename T>
__device__ __forceinline__ void widen_int8(uint32_t w, uint32_t& lo, uint32_t& hi);
template <>
__device__ __forceinline__ void widen_int8<__half>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 c = __half2half2(__ushort_as_half(0x6480));  // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), c);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), c);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}
template <>
__device__ __forceinline__ void widen_int8<__nv_bfloat16>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
  const uint32_t a0 = a & 0xff7fff7fu, a1 = a & 0xff80ff80u, b0 = b & 0xff7fff7fu, b1 = b & 0xff80ff80u;
  const __nv_bfloat162 x =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a0), *reinterpret_cast<const __nv_bfloat162*>(&a1));
  const __nv_bfloat162 y =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b0), *reinterpret_cast<const __nv_bfloat162*>(&b1));
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

// Two e4m3 codes (the low 16 bits of w) as a 16-bit pair, exactly (every e4m3 value is an fp16 and a bf16 value).
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
template <typename T>
__device__ __forceinline__ void widen_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = e4m3x2_f16x2(w & 0xffffu);
  hi = e4m3x2_f16x2(w >> 16);
  if constexpr (!std::is_same<T, __half>::value) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = pack_h2<T>(a.x, a.y);
    hi = pack_h2<T>(b.x, b.y);
  }
}
template <typename T, int KIND>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == B2P_KV_INT8)
    widen_int8<T>(w, lo, hi);
  else
    widen_e4m3<T>(w, lo, hi);
}

}  // namespace b2p
