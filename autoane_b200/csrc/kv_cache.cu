// kv_cache.cu — writing new tokens' keys and values into a paged cache (rotary
// positions and 8-bit quantisation in the same pass) and reading them back.
//
// A vector of 64 channels (one token, one head) belongs to 8 lanes, 8 channels
// each: one 16-byte load, the largest |x| by three shuffles, one 8-byte (codes)
// or 16-byte store. The partner channels of a half-split rotation are in lane
// +- rot/16 and come by shuffles of the 16-bit pairs as loaded. A warp has
// four tokens and goes through their heads together, so that it need not diverge
// between Q, K and V and loads a token's angles once.
// Bound: the reads and writes. 65536 tokens of 15 / 5 heads to int8: append 380 MB in
// 69 us (5.5 TB/s), read back 131 MB in 23 us (5.6 TB/s, part of it L2's).
#include <cstdint>
#include "decode.cuh"
#include "ptx.cuh"

namespace b2p {

int kv_view(const b2p_kv_cache* c, int dtype, KvView* out) {
  B2P_REQUIRE(c, "null cache");
  B2P_REQUIRE(dtype == B2P_F16 || dtype == B2P_BF16, "dtype must be B2P_F16 or B2P_BF16");
  B2P_REQUIRE(c->kind == B2P_KV_16 || c->kind == B2P_KV_INT8 || c->kind == B2P_KV_E4M3,
              "cache kind must be B2P_KV_16, B2P_KV_INT8 or B2P_KV_E4M3");
  B2P_REQUIRE(c->k && c->v, "null cache buffer");
  B2P_REQUIRE(c->page_size >= 8 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
              "page_size must be a power of two from 8 to 1024 (got %d)", c->page_size);
  B2P_REQUIRE(c->n_pages >= 1 && c->kv_heads >= 1, "n_pages and kv_heads must be positive");
  B2P_REQUIRE((long long)c->n_pages * c->page_size < (1ll << 31), "n_pages * page_size must be below 2^31");
  B2P_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u) == 0,
              "cache buffers must be 16-byte aligned");
  if (c->kind != B2P_KV_16) {
    B2P_REQUIRE(c->k_scale && c->v_scale, "8-bit caches need k_scale and v_scale");
    B2P_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 7u) == 0,
                "cache scales must be 8-byte aligned");
  }
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->n_pages = c->n_pages;
  out->page_shift = shift;
  out->kv_heads = c->kv_heads;
  out->kind = c->kind;
  return B2P_OK;
}

namespace {

constexpr int kKvThreads = 256;

struct AppendArgs {
  KvView c;
  const void* qkv;
  void* q_out;
  const int32_t* slots;
  const int32_t* positions;
  const float* rope;
  long long ld_qkv, ld_q;
  int heads, max_pos, rot, interleaved, n_tokens;
};

// fmaxf that keeps a NaN: a vector with one reads back as NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {  // a in the low byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Four values of at most 127.5 as int8, rounded to nearest even: above 2^23 a sum's low byte is the integer.
__device__ __forceinline__ uint32_t int8x4(const float* y) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(__fadd_rn(y[i], 12582912.f));
  return __byte_perm(__byte_perm(v[0], v[1], 0x0040), __byte_perm(v[2], v[3], 0x0040), 0x5410);
}

enum RopeMode { ROPE_NONE, ROPE_HALVES, ROPE_PAIRS };

// A warp takes every head of four tokens, four at a time with the next four on their way; or, where calls are small
// (ONE), one head: the tokens' heads are then spread over more warps.
template <typename T, int KIND, int MODE, bool ONE>
__global__ void __launch_bounds__(kKvThreads) kv_append_kernel(AppendArgs a, uint32_t* status) {
  constexpr int HC = ONE ? 1 : 4;
  pdl_enter();
  const int kv = a.c.kv_heads, rotated = a.heads + kv, total = rotated + kv;
  const int warp = (int)(((long long)blockIdx.x * kKvThreads + threadIdx.x) >> 5);
  const int lane = threadIdx.x & 31, l = lane & 7;
  const int first = ONE ? warp % total : 0, end = ONE ? first + 1 : total;
  const int t = (ONE ? warp / total : warp) * 4 + (lane >> 3);
  const bool live = t < a.n_tokens;

  const T* row = static_cast<const T*>(a.qkv) + (live ? t : 0) * a.ld_qkv + l * 8;
  auto load = [&](int h, uint4 (&raw)[HC]) {
#pragma unroll
    for (int i = 0; i < HC; ++i)
      raw[i] = h + i < end ? __ldcs(reinterpret_cast<const uint4*>(row + (h + i) * kKvHeadDim)) : make_uint4(0, 0, 0, 0);
  };
  uint4 raw[HC];
  load(first, raw);
  long long at0 = -1;  // vector of the token's slot, KV head 0
  if (live && end > a.heads) {
    const int slot = a.slots[t];
    if (slot >= (a.c.n_pages << a.c.page_shift))
      atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
    else if (slot >= 0)
      at0 = a.c.vec(slot >> a.c.page_shift, 0, slot & ((1 << a.c.page_shift) - 1));
  }
  // this lane's angles: channel j becomes x_j c_j + p_j s_j with p_j its partner channel, s_j negative for
  // the first of a pair; outside the rotated part c = 1 and p = s = 0
  const bool turns = l * 8 < a.rot;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    c[e] = 1.f;
    s[e] = 0.f;
  }
  int partner = lane;
  if (MODE != ROPE_NONE && first < rotated) {
    int pos = live ? a.positions[t] : 0;
    if (pos < 0 || pos >= a.max_pos) {
      atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
      pos = 0;
    }
    const float4* tab = reinterpret_cast<const float4*>(a.rope + (long long)pos * a.rot);
    if (turns && MODE == ROPE_PAIRS) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 w = tab[l * 2 + i];
        c[4 * i] = c[4 * i + 1] = w.x;
        c[4 * i + 2] = c[4 * i + 3] = w.z;
        s[4 * i] = -w.y;
        s[4 * i + 1] = w.y;
        s[4 * i + 2] = -w.w;
        s[4 * i + 3] = w.w;
      }
    } else if (turns) {
      const int half_lanes = a.rot >> 4;  // lanes of one half of the rotated part
      const bool second = l >= half_lanes;
      partner = second ? lane - half_lanes : lane + half_lanes;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 w = tab[(second ? l - half_lanes : l) * 4 + i];
        c[2 * i] = w.x;
        c[2 * i + 1] = w.z;
        s[2 * i] = second ? w.y : -w.y;
        s[2 * i + 1] = second ? w.w : -w.w;
      }
    }
  }

  T* q_out = static_cast<T*>(a.q_out) + (live ? t : 0) * a.ld_q + l * 8;
#pragma unroll 1
  for (int h0 = first; h0 < end; h0 += HC) {
    uint4 next[HC];
    if (!ONE) load(h0 + HC, next);
#pragma unroll
    for (int i = 0; i < HC; ++i) {
      const int h = h0 + i;  // (the same in all lanes)
      if (h >= end) break;
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = H2<T>::to_f2(*reinterpret_cast<const typename H2<T>::V*>(&w[e]));
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
      }
      if (MODE != ROPE_NONE && h < rotated) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t o = MODE == ROPE_PAIRS ? __byte_perm(w[e], 0, 0x1032) : __shfl_sync(~0u, w[e], partner);
          if (!turns) o = 0;
          const float2 f = H2<T>::to_f2(*reinterpret_cast<typename H2<T>::V*>(&o));
          x[2 * e] = x[2 * e] * c[2 * e] + f.x * s[2 * e];
          x[2 * e + 1] = x[2 * e + 1] * c[2 * e + 1] + f.y * s[2 * e + 1];
        }
      }
      if (h < a.heads) {
        if (live)
          *reinterpret_cast<uint4*>(q_out + h * kKvHeadDim) = make_uint4(
              pack_h2<T>(x[0], x[1]), pack_h2<T>(x[2], x[3]), pack_h2<T>(x[4], x[5]), pack_h2<T>(x[6], x[7]));
        continue;
      }
      const bool is_v = h >= rotated;
      const long long at = at0 + ((long long)(h - (is_v ? rotated : a.heads)) << a.c.page_shift);
      uint8_t* codes = is_v ? a.c.v : a.c.k;
      if (KIND == B2P_KV_16) {
        if (at0 >= 0)
          *reinterpret_cast<uint4*>(codes + at * 128 + l * 16) = make_uint4(
              pack_h2<T>(x[0], x[1]), pack_h2<T>(x[2], x[3]), pack_h2<T>(x[4], x[5]), pack_h2<T>(x[6], x[7]));
      } else {
        float top = max_nan(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
        for (int e = 2; e < 8; ++e) top = max_nan(top, fabsf(x[e]));
        for (int o = 1; o < 8; o <<= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
        top = max_nan(top, 1e-30f);
        constexpr float kTop = KIND == B2P_KV_INT8 ? 127.f : 448.f;
        const float inv = __fmul_rn(__frcp_rn(top), kTop);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], inv);
        uint2 o;
        if (KIND == B2P_KV_INT8)
          o = make_uint2(int8x4(x), int8x4(x + 4));
        else
          o = make_uint2(e4m3_pair(x[0], x[1]) | e4m3_pair(x[2], x[3]) << 16,
                         e4m3_pair(x[4], x[5]) | e4m3_pair(x[6], x[7]) << 16);
        if (at0 >= 0) {
          *reinterpret_cast<uint2*>(codes + at * 64 + l * 8) = o;
          // (an infinite value's vector too has a NaN scale: its codes are 0 and, for int8, no NaN can be one)
          if (l == 0)
            (is_v ? a.c.v_scale : a.c.k_scale)[at] = top < INFINITY ? top * (1.0f / kTop) : __int_as_float(0x7fc00000);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < HC; ++i) raw[i] = next[i];
  }
}

struct ReadArgs {
  KvView c;
  const int32_t* slots;
  void* k_out;
  void* v_out;
  long long ld_k, ld_v;
  int n_tokens;
};

// K and V of one token and KV head by 8 lanes.
template <typename T, int KIND>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(ReadArgs a, uint32_t* status) {
  pdl_enter();
  const long long group = ((long long)blockIdx.x * kKvThreads + threadIdx.x) >> 3;
  const int l = threadIdx.x & 7;
  if (group >= (long long)a.n_tokens * a.c.kv_heads) return;
  const int t = (int)(group / a.c.kv_heads), kvh = (int)(group - (long long)t * a.c.kv_heads);
  int slot = a.slots[t];
  if (slot >= (a.c.n_pages << a.c.page_shift)) {
    atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
    slot = -1;
  }
  uint4 r[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (slot >= 0) {
    const long long at = a.c.vec(slot >> a.c.page_shift, kvh, slot & ((1 << a.c.page_shift) - 1));
    if (KIND == B2P_KV_16) {
      r[0] = *reinterpret_cast<const uint4*>(a.c.k + at * 128 + l * 16);
      r[1] = *reinterpret_cast<const uint4*>(a.c.v + at * 128 + l * 16);
    } else {
      const uint2 w[2] = {*reinterpret_cast<const uint2*>(a.c.k + at * 64 + l * 8),
                          *reinterpret_cast<const uint2*>(a.c.v + at * 64 + l * 8)};
      const float scale[2] = {a.c.k_scale[at], a.c.v_scale[at]};
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint32_t p[4];
        widen4<T, KIND>(w[v].x, p[0], p[1]);
        widen4<T, KIND>(w[v].y, p[2], p[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = H2<T>::to_f2(*reinterpret_cast<typename H2<T>::V*>(&p[e]));
          p[e] = pack_h2<T>(f.x * scale[v], f.y * scale[v]);
        }
        r[v] = make_uint4(p[0], p[1], p[2], p[3]);
      }
    }
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + (long long)t * a.ld_k + kvh * kKvHeadDim + l * 8) = r[0];
  *reinterpret_cast<uint4*>(static_cast<T*>(a.v_out) + (long long)t * a.ld_v + kvh * kKvHeadDim + l * 8) = r[1];
}

template <typename T, int KIND, int MODE>
int append_mode(const AppendArgs& a, const DeviceCtx* c, cudaStream_t st) {
  // One head a warp while that does not fill the GPU four times over: a warp that goes through 25 heads takes longer
  // than the whole call of a few tokens. Measured, 25 heads, one a warp / all: 8 tokens 1.8 / 6.2 us, 2051 5.0 / 7.4,
  // 4096 8.3 / 10.2, 8192 14.7 / 11.3, 16384 32 / 19.
  const int total = a.heads + 2 * a.c.kv_heads;
  const long long quads = ((long long)a.n_tokens + 3) / 4;
  const bool one = quads * total <= (long long)c->num_sms * 64 * 4;
  const long long blocks = (quads * (one ? total : 1) * 32 + kKvThreads - 1) / kKvThreads;
  B2P_CHECK_CUDA(launch_pdl(one ? kv_append_kernel<T, KIND, MODE, true> : kv_append_kernel<T, KIND, MODE, false>,
                            dim3((unsigned)blocks), dim3(kKvThreads), 0, st, a, c->status));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

template <typename T, int KIND>
int append_t(const AppendArgs& a, const DeviceCtx* c, cudaStream_t st) {
  if (!a.rot) return append_mode<T, KIND, ROPE_NONE>(a, c, st);
  return a.interleaved ? append_mode<T, KIND, ROPE_PAIRS>(a, c, st) : append_mode<T, KIND, ROPE_HALVES>(a, c, st);
}

template <typename T, int KIND>
int read_t(const ReadArgs& a, const DeviceCtx* c, cudaStream_t st) {
  const long long threads = (long long)a.n_tokens * a.c.kv_heads * 8;
  const long long blocks = (threads + kKvThreads - 1) / kKvThreads;
  B2P_REQUIRE(blocks < (1ll << 31), "too many tokens in one call");
  B2P_CHECK_CUDA(
      launch_pdl(kv_read_kernel<T, KIND>, dim3((unsigned)blocks), dim3(kKvThreads), 0, st, a, c->status));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

int check_rows(const void* p, int ld, int cols, const char* name) {
  B2P_REQUIRE(p, "null %s", name);
  B2P_REQUIRE(ld >= cols && ld % 8 == 0, "%s rows must hold %d columns and keep 16-byte alignment (pitch %d)", name,
              cols, ld);
  B2P_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15u) == 0, "%s must be 16-byte aligned", name);
  return B2P_OK;
}

}  // namespace
}  // namespace b2p

using namespace b2p;

extern "C" {

int b2p_kv_append(const b2p_kv_cache* cache, const void* qkv, int ld_qkv, int heads, void* q_out, int ld_q,
                  const int32_t* slots, const int32_t* positions, const float* rope, int max_pos, int rot,
                  int interleaved, int n_tokens, int dtype, void* stream) {
  AppendArgs a;
  int rc = kv_view(cache, dtype, &a.c);
  if (rc) return rc;
  B2P_REQUIRE(n_tokens >= 0, "n_tokens must not be negative");
  B2P_REQUIRE(heads >= 1 && heads <= 4096 && a.c.kv_heads <= 4096, "heads must be from 1 to 4096");
  B2P_REQUIRE(rot >= 0 && rot <= kKvHeadDim && rot % 16 == 0, "rot must be 0, 16, 32, 48 or 64 (got %d)", rot);
  if (n_tokens == 0) return B2P_OK;
  if ((rc = check_rows(qkv, ld_qkv, (heads + 2 * a.c.kv_heads) * kKvHeadDim, "qkv"))) return rc;
  if ((rc = check_rows(q_out, ld_q, heads * kKvHeadDim, "q_out"))) return rc;
  B2P_REQUIRE(slots, "null slots");
  if (rot) {
    B2P_REQUIRE(rope && positions && max_pos >= 1, "rotation needs rope, positions and max_pos");
    B2P_REQUIRE((reinterpret_cast<uintptr_t>(rope) & 15u) == 0, "rope must be 16-byte aligned");
  }
  DeviceCtx* c = nullptr;
  if ((rc = ctx_get(&c))) return rc;
  a.qkv = qkv;
  a.q_out = q_out;
  a.slots = slots;
  a.positions = positions;
  a.rope = rope;
  a.ld_qkv = ld_qkv;
  a.ld_q = ld_q;
  a.heads = heads;
  a.max_pos = max_pos;
  a.rot = rot;
  a.interleaved = interleaved != 0;
  a.n_tokens = n_tokens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == B2P_BF16;
  switch (a.c.kind) {
    case B2P_KV_INT8:
      return bf ? append_t<__nv_bfloat16, B2P_KV_INT8>(a, c, st) : append_t<__half, B2P_KV_INT8>(a, c, st);
    case B2P_KV_E4M3:
      return bf ? append_t<__nv_bfloat16, B2P_KV_E4M3>(a, c, st) : append_t<__half, B2P_KV_E4M3>(a, c, st);
    default:
      return bf ? append_t<__nv_bfloat16, B2P_KV_16>(a, c, st) : append_t<__half, B2P_KV_16>(a, c, st);
  }
}

int b2p_kv_read(const b2p_kv_cache* cache, const int32_t* slots, int n_tokens, void* k_out, int ld_k, void* v_out,
                int ld_v, int dtype, void* stream) {
  ReadArgs a;
  int rc = kv_view(cache, dtype, &a.c);
  if (rc) return rc;
  B2P_REQUIRE(n_tokens >= 0, "n_tokens must not be negative");
  B2P_REQUIRE(a.c.kv_heads <= 4096, "kv_heads must be at most 4096");
  if (n_tokens == 0) return B2P_OK;
  if ((rc = check_rows(k_out, ld_k, a.c.kv_heads * kKvHeadDim, "k_out"))) return rc;
  if ((rc = check_rows(v_out, ld_v, a.c.kv_heads * kKvHeadDim, "v_out"))) return rc;
  B2P_REQUIRE(slots, "null slots");
  DeviceCtx* c = nullptr;
  if ((rc = ctx_get(&c))) return rc;
  a.slots = slots;
  a.k_out = k_out;
  a.v_out = v_out;
  a.ld_k = ld_k;
  a.ld_v = ld_v;
  a.n_tokens = n_tokens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == B2P_BF16;
  switch (a.c.kind) {
    case B2P_KV_INT8:
      return bf ? read_t<__nv_bfloat16, B2P_KV_INT8>(a, c, st) : read_t<__half, B2P_KV_INT8>(a, c, st);
    case B2P_KV_E4M3:
      return bf ? read_t<__nv_bfloat16, B2P_KV_E4M3>(a, c, st) : read_t<__half, B2P_KV_E4M3>(a, c, st);
    default:
      return bf ? read_t<__nv_bfloat16, B2P_KV_16>(a, c, st) : read_t<__half, B2P_KV_16>(a, c, st);
  }
}

}  // extern "C"
