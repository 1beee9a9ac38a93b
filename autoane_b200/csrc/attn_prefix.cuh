// attn_prefix.cuh — the work division of attention over a shared prefix,
// common to its kernels (attn_prefix.cu, attn_prefix_tc.cu).
#pragma once
#include "decode.cuh"

namespace b2p {

// Rows of one KV head: r = (b * q_len + i) * group + g, for query i of sequence b and query head
// kvh * group + g. A part is what one kernel block computes for some rows over some keys: the rows'
// maximum score (log2 domain), sum of exponentials and unnormalised output. The first parts split the
// prefix, those from max(n_prefix, n_last) on each sequence's suffix, every split a fixed number of keys.
// attn_join_kernel joins a row's parts.
struct PrefixSplit {
  int pair_rows;               // rows below it: n_prefix parts of prefix_chunk keys
  int n_prefix, prefix_chunk;
  int n_last, last_chunk;      // rows from it on: n_last parts of last_chunk keys
};

struct PrefixArgs : PrefixSplit {
  KvView c;
  const void* q;
  void* out;
  float* lse;
  const int32_t* prefix_pages;
  const int32_t* suffix_pages;
  const int32_t* suffix_lens;
  float* part_o;    // [part][kv_heads * rows][64]
  float2* part_ml;  // [part][kv_heads * rows] (maximum, sum)
  long long ld_q, ld_out;
  int batch, q_len, group, rows;  // rows = batch * q_len * group, of one KV head
  int prefix_len, suffix_pitch, max_suffix;
  int suffix_part;             // first part of a suffix
  int n_suffix, suffix_chunk;  // suffix parts and keys of each
};

// The prefix part on the tcgen05 tensor cores (attn_prefix_tc.cu), and its division of the prefix.
int launch_prefix_tc(const PrefixArgs& a, bool bf16, cudaStream_t st);
void prefix_tc_plan(int rows, int kv_heads, int prefix_len, PrefixSplit* s);

constexpr int kTcStageKeys = 128;  // its parts are multiples of this many keys
constexpr int kSms = 148;  // of a B200: what the work divisions aim at
constexpr float kScaleLog2 = 0.125f * 1.4426950408889634f;  // 1/sqrt(64) * log2(e)

// The length of sequence b's suffix (a bad entry counts as empty and is recorded).
__device__ __forceinline__ int suffix_len(const PrefixArgs& a, int b, uint32_t* status) {
  const int n = a.suffix_lens[b];
  if (n < 0 || n > a.max_suffix) {
    atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
    return 0;
  }
  return n;
}

// Parts of row r of a KV head, its suffix holding `len` tokens.
__device__ __forceinline__ int parts_of(const PrefixArgs& a, int r, int len) {
  return (r < a.pair_rows ? a.n_prefix : a.n_last) + (len + a.suffix_chunk - 1) / a.suffix_chunk;
}

__device__ __forceinline__ float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Join the parts of row r of KV head kvh and write the output, by the 16 threads of a half warp (sub = 0..15). The
// order of the parts is fixed, whoever joins them.
template <typename T>
__device__ __forceinline__ void join_row(const PrefixArgs& a, int kvh, int r, int len, int sub) {
  const unsigned half = 0xffffu << (threadIdx.x & 16);
  const int shared = r < a.pair_rows ? a.n_prefix : a.n_last;
  const int parts = parts_of(a, r, len);
  const long long stride = (long long)a.c.kv_heads * a.rows, at0 = (long long)kvh * a.rows + r;
  auto slot = [&](int p) { return (p < shared ? p : p - shared + a.suffix_part) * stride + at0; };
  float top = -INFINITY;
  float2 ml = make_float2(-INFINITY, 0.f);
  for (int p0 = 0; p0 < parts; p0 += 16) {
    if (p0 + sub < parts) {
      ml = __ldcg(a.part_ml + slot(p0 + sub));
      top = fmaxf(top, ml.x);
    }
  }
  for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(half, top, o));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += 16) {
    if (parts > 16) ml = p0 + sub < parts ? __ldcg(a.part_ml + slot(p0 + sub)) : make_float2(-INFINITY, 0.f);
    const float f = exp2_sfu(ml.x - ref);
    float part_sum = f * ml.y;
    for (int o = 8; o; o >>= 1) part_sum += __shfl_xor_sync(half, part_sum, o);
    sum += part_sum;
    const int n = min(16, parts - p0);
    for (int k0 = 0; k0 < n; k0 += 8) {  // eight loads in flight
      float4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < n) x[k] = __ldcg(reinterpret_cast<const float4*>(a.part_o + slot(p0 + k0 + k) * kKvHeadDim) + sub);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(half, f, k0 + k, 16);
        if (k0 + k < n) {
          acc.x += w * x[k].x;
          acc.y += w * x[k].y;
          acc.z += w * x[k].z;
          acc.w += w * x[k].w;
        }
      }
    }
  }
  // (a row that sees nothing has no weights; one whose scores are all NaN has no maximum either, but its sum is NaN)
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int token = r / a.group, h = kvh * a.group + r % a.group;
  T* out = static_cast<T*>(a.out) + (long long)token * a.ld_out + h * kKvHeadDim + sub * 4;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_h2<T>(acc.x * inv, acc.y * inv), pack_h2<T>(acc.z * inv, acc.w * inv));
  if (a.lse && sub == 0)
    a.lse[(long long)token * a.c.kv_heads * a.group + h] = sum == 0.f ? -INFINITY : ref + log2f(sum);
}

}  // namespace b2p
