// attn_prefix.cuh — the work division of attention over a shared prefix,
// common to its kernels (attn_prefix.cu, attn_prefix_tc.cu).
#pragma once
#include "decode.cuh"

namespace b2p {

// Rows of one KV head: r = (b * q_len + i) * group + g, for query i of sequence b and query head
// kvh * group + g. A part is what one kernel block computes for some rows over some keys: the rows'
// maximum score (log2 domain), sum of exponentials and unnormalised output. The first parts split the
// prefix, those from max(n_prefix, n_last) on each sequence's suffix, every split a fixed number of keys.
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

}  // namespace b2p
