// kv_cache.cu — writing new tokens' keys and values into a paged cache (rotary
// positions and 8-bit quantisation in the same pass) and reading them back.
//
// A vector of 64 channels (one token, one head) belongs to 8 lanes, 8 channels
// each: one 16-byte load, the largest |x| by three shuffles, one 8-byte (codes)
// or 16-byte store. The partner channels of a half-split rotation are in lane
// +- rot/16 and come by shuffles of the 16-bit pairs as loaded.
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

template <typename T, int KIND, int HC>
__global__ void __launch_bounds__(kKvThreads) kv_append_kernel(AppendArgs a, uint32_t* status) {
  pdl_enter();
  const int total = a.heads + 2 * a.c.kv_heads;
  const int chunks = (total + HC - 1) / HC;
  const long long group = ((long long)blockIdx.x * kKvThreads + threadIdx.x) >> 3;
  const int l = threadIdx.x & 7;
  const bool live = group < (long long)a.n_tokens * chunks;
  const int t = live ? (int)(group / chunks) : 0;
  const int h0 = live ? (int)(group % chunks) * HC : 0;

  const T* row = static_cast<const T*>(a.qkv) + (long long)t * a.ld_qkv;
  uint4 raw[HC];
#pragma unroll
  for (int i = 0; i < HC; ++i)
    raw[i] = (live && h0 + i < total) ? *reinterpret_cast<const uint4*>(row + (h0 + i) * kKvHeadDim + l * 8)
                                      : make_uint4(0, 0, 0, 0);
  int slot = -1;
  if (live && h0 + HC > a.heads) {
    slot = a.slots[t];
    if (slot >= (a.c.n_pages << a.c.page_shift)) {
      atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
      slot = -1;
    }
  }
  // this lane's angles: channel j becomes x_j c_j + p_j s_j with p_j its partner channel, s_j negative for
  // the first of a pair
  const bool turns = l * 8 < a.rot;
  const int half_lanes = a.rot >> 4;  // lanes of one half of the rotated part
  float c[8], s[8];
  if (a.rot && h0 < a.heads + a.c.kv_heads) {
    int pos = live ? a.positions[t] : 0;
    if (pos < 0 || pos >= a.max_pos) {
      if (live) atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
      pos = 0;
    }
    const float4* tab = reinterpret_cast<const float4*>(a.rope + (long long)pos * a.rot);
    if (turns) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 w = __ldg(tab + l * 2 + i);
          c[4 * i] = c[4 * i + 1] = w.x;
          c[4 * i + 2] = c[4 * i + 3] = w.z;
          s[4 * i] = -w.y;
          s[4 * i + 1] = w.y;
          s[4 * i + 2] = -w.w;
          s[4 * i + 3] = w.w;
        }
      } else {
        const bool second = l >= half_lanes;
        const int l0 = second ? l - half_lanes : l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 w = __ldg(tab + l0 * 4 + i);
          c[2 * i] = w.x;
          c[2 * i + 1] = w.z;
          s[2 * i] = second ? w.y : -w.y;
          s[2 * i + 1] = second ? w.w : -w.w;
        }
      }
    }
  }
  const int lane = threadIdx.x & 31;
  const int partner = !turns ? lane : a.interleaved ? lane : l >= half_lanes ? lane - half_lanes : lane + half_lanes;

#pragma unroll
  for (int i = 0; i < HC; ++i) {
    const int h = h0 + i;
    uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = H2<T>::to_f2(*reinterpret_cast<typename H2<T>::V*>(&w[e]));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
    if (a.rot) {  // every lane shuffles; a vector that does not turn keeps its channels
      float p[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t o = __shfl_sync(~0u, w[e], partner);
        const float2 f = H2<T>::to_f2(*reinterpret_cast<typename H2<T>::V*>(&o));
        p[2 * e] = a.interleaved ? f.y : f.x;
        p[2 * e + 1] = a.interleaved ? f.x : f.y;
      }
      if (turns && h < a.heads + a.c.kv_heads) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * c[e] + p[e] * s[e];
      }
    }
    if (live && h < a.heads) {
      T* q = static_cast<T*>(a.q_out) + (long long)t * a.ld_q + h * kKvHeadDim + l * 8;
      *reinterpret_cast<uint4*>(q) = make_uint4(pack_h2<T>(x[0], x[1]), pack_h2<T>(x[2], x[3]), pack_h2<T>(x[4], x[5]),
                                                pack_h2<T>(x[6], x[7]));
    }
    float top = 0.f;
    if (KIND != B2P_KV_16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(x[e]));
      for (int o = 1; o < 8; o <<= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
      top = max_nan(top, 1e-30f);
    }
    if (h < a.heads || h >= total || slot < 0) continue;
    const bool is_v = h >= a.heads + a.c.kv_heads;
    const int kvh = h - a.heads - (is_v ? a.c.kv_heads : 0);
    const long long at = a.c.vec(slot >> a.c.page_shift, kvh, slot & ((1 << a.c.page_shift) - 1));
    uint8_t* codes = is_v ? a.c.v : a.c.k;
    if (KIND == B2P_KV_16) {
      *reinterpret_cast<uint4*>(codes + at * 128 + l * 16) = make_uint4(
          pack_h2<T>(x[0], x[1]), pack_h2<T>(x[2], x[3]), pack_h2<T>(x[4], x[5]), pack_h2<T>(x[6], x[7]));
    } else {
      constexpr float kTop = KIND == B2P_KV_INT8 ? 127.f : 448.f;
      const float inv = __fmul_rn(__frcp_rn(top), kTop);
      uint32_t o[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float* y = x + 4 * e;
        if (KIND == B2P_KV_INT8) {
          const int a0 = __float2int_rn(y[0] * inv), a1 = __float2int_rn(y[1] * inv);
          const int a2 = __float2int_rn(y[2] * inv), a3 = __float2int_rn(y[3] * inv);
          o[e] = (uint32_t)(a0 & 255) | (uint32_t)(a1 & 255) << 8 | (uint32_t)(a2 & 255) << 16 | (uint32_t)a3 << 24;
        } else {
          o[e] = e4m3_pair(y[0] * inv, y[1] * inv) | e4m3_pair(y[2] * inv, y[3] * inv) << 16;
        }
      }
      *reinterpret_cast<uint2*>(codes + at * 64 + l * 8) = make_uint2(o[0], o[1]);
      if (l == 0) (is_v ? a.c.v_scale : a.c.k_scale)[at] = top * (1.0f / kTop);
    }
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

template <typename T, int KIND>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(ReadArgs a, uint32_t* status) {
  pdl_enter();
  const int per = 2 * a.c.kv_heads;
  const long long group = ((long long)blockIdx.x * kKvThreads + threadIdx.x) >> 3;
  const int l = threadIdx.x & 7;
  if (group >= (long long)a.n_tokens * per) return;
  const int t = (int)(group / per);
  const int h = (int)(group % per);
  const bool is_v = h >= a.c.kv_heads;
  const int kvh = is_v ? h - a.c.kv_heads : h;
  int slot = a.slots[t];
  if (slot >= (a.c.n_pages << a.c.page_shift)) {
    atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
    slot = -1;
  }
  uint4 r = make_uint4(0, 0, 0, 0);
  if (slot >= 0) {
    const long long at = a.c.vec(slot >> a.c.page_shift, kvh, slot & ((1 << a.c.page_shift) - 1));
    const uint8_t* codes = is_v ? a.c.v : a.c.k;
    if (KIND == B2P_KV_16) {
      r = *reinterpret_cast<const uint4*>(codes + at * 128 + l * 16);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + at * 64 + l * 8);
      const float scale = (is_v ? a.c.v_scale : a.c.k_scale)[at];
      uint32_t p[4];
      widen4<T, KIND>(w.x, p[0], p[1]);
      widen4<T, KIND>(w.y, p[2], p[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = H2<T>::to_f2(*reinterpret_cast<typename H2<T>::V*>(&p[e]));
        p[e] = pack_h2<T>(f.x * scale, f.y * scale);
      }
      r = make_uint4(p[0], p[1], p[2], p[3]);
    }
  }
  T* out = is_v ? static_cast<T*>(a.v_out) + (long long)t * a.ld_v : static_cast<T*>(a.k_out) + (long long)t * a.ld_k;
  *reinterpret_cast<uint4*>(out + kvh * kKvHeadDim + l * 8) = r;
}

template <typename T, int KIND>
int append_t(const AppendArgs& a, const DeviceCtx* c, cudaStream_t st) {
  // One head per lane group while the call does not fill the GPU (latency), four heads of a token
  // otherwise: a token's angles are then loaded once for four heads.
  const int total = a.heads + 2 * a.c.kv_heads;
  const bool few = (long long)a.n_tokens * total * 8 <= (long long)c->num_sms * 2048;
  const int hc = few ? 1 : 4;
  const long long threads = (long long)a.n_tokens * ((total + hc - 1) / hc) * 8;
  const long long blocks = (threads + kKvThreads - 1) / kKvThreads;
  B2P_REQUIRE(blocks < (1ll << 31), "too many tokens in one call");
  B2P_CHECK_CUDA(launch_pdl(few ? kv_append_kernel<T, KIND, 1> : kv_append_kernel<T, KIND, 4>, dim3((unsigned)blocks),
                            dim3(kKvThreads), 0, st, a, c->status));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

template <typename T, int KIND>
int read_t(const ReadArgs& a, const DeviceCtx* c, cudaStream_t st) {
  const long long threads = (long long)a.n_tokens * 2 * a.c.kv_heads * 8;
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
