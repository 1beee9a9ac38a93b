// sample.cu — sampling a token per row of logits with temperature, top-k, top-p
// and min-p, from given uniform numbers.
//
// A token's weight is an integer, w = round(2^31 · 2^-depth), its depth below
// the row's maximum taken in steps of 2^-20 (a key of at most 26 bits), so every
// sum is exact in 64 bits whatever its order: the filters and the draw are the
// same in every run. The kept tokens are a prefix of the ranking by (key, index),
// so each filter is a cut: a key and how many of the tokens with just that key
// stay. top-k's cut is found by counts, top-p's by weights, both in a histogram
// over the upper key bits that is refined in the bin where the cut lies.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "engine.cuh"
#include "ptx.cuh"

namespace b2p {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr float kDeep = 64.f;            // depths are cut here
constexpr float kSteps = 1048576.f;      // key steps per unit of depth
constexpr uint32_t kLive = 32u << 20;    // keys above it weigh nothing: 2^31 · 2^-32 rounds to 0
constexpr int kBins = 1024;              // of the histogram's first two levels; the third has 32

struct SampleArgs {
  const void* logits;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  float* logprobs;
  long long ld;
  int vocab;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Depth of a logit x below the maximum m as a key; c = log2(e) / T.
__device__ __forceinline__ uint32_t key_of(float x, float m, float c) {
  // m - x is NaN for m = x = inf (depth 0) and for a NaN logit (deepest)
  const float d = x == m ? 0.f : __fmul_rn(m - x, c);
  return __float2uint_rn(d < kDeep ? d * kSteps : kDeep * kSteps);
}
__device__ __forceinline__ unsigned long long weight_of(uint32_t key) {
  if (key > kLive) return 0;
  return __float2ull_rn(exp2f(-(float)key * (1.f / kSteps)) * 2147483648.f);
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V x, V* scratch, Op op) {
  for (int o = 16; o; o >>= 1) x = op(x, __shfl_xor_sync(~0u, x, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  x = scratch[threadIdx.x & 31];
  for (int o = 16; o; o >>= 1) x = op(x, __shfl_xor_sync(~0u, x, o));
  return x;
}

struct Cut {
  uint32_t key;   // tokens with a smaller key stay
  uint32_t ties;  // and this many, in index order, of those with just this key
};

struct Smem {
  unsigned long long weight[kBins];
  uint32_t count[kBins];
  unsigned long long scratch64[32];
  float scratchf[32];
  uint32_t bin;
  unsigned long long below_w, below_c;
};

// The first bin at which the running measure (counts, or weights) reaches `aim`; s.bin = kBins when none does.
// Every thread owns one bin. below_c / below_w receive the sums before the bin.
__device__ __forceinline__ void find_bin(Smem& s, bool by_count, double aim, unsigned long long c0,
                                         unsigned long long w0, int bins) {
  const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
  const unsigned long long c = i < bins ? s.count[i] : 0, w = i < bins ? s.weight[i] : 0;
  unsigned long long ic = c, iw = w;
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long pc = __shfl_up_sync(~0u, ic, o), pw = __shfl_up_sync(~0u, iw, o);
    if (lane >= o) {
      ic += pc;
      iw += pw;
    }
  }
  __shared__ unsigned long long sc[kWarps], sw[kWarps];
  __syncthreads();
  if (lane == 31) {
    sc[warp] = ic;
    sw[warp] = iw;
  }
  if (i == 0) s.bin = kBins;
  __syncthreads();
  unsigned long long bc = c0, bw = w0;
  for (int k = 0; k < warp; ++k) {
    bc += sc[k];
    bw += sw[k];
  }
  ic += bc;
  iw += bw;
  const double before = by_count ? (double)(ic - c) : (double)(iw - w);
  const double after = by_count ? (double)ic : (double)iw;
  if (c && before < aim && after >= aim) {  // one bin at most: the measure does not fall
    s.bin = i;
    s.below_c = ic - c;
    s.below_w = iw - w;
  }
  __syncthreads();
}

template <typename T>
struct Row {
  const T* x;
  int vocab;
  float m, c;
  __device__ __forceinline__ uint32_t key(int j) const { return key_of(to_float(x[j]), m, c); }
};

// The cut at which the measure reaches `aim` (> 0), starting from the first-level histogram in s.
// With the whole row below it: {kLive + 1, 0}. below_w: the weight of what the cut keeps.
template <typename T>
__device__ Cut find_cut(Smem& s, const Row<T>& row, bool by_count, double aim, unsigned long long& kept_w) {
  unsigned long long c0 = 0, w0 = 0;
  find_bin(s, by_count, aim, 0, 0, kBins);
  uint32_t prefix = s.bin;
  if (prefix == kBins) {
    kept_w = ~0ull;
    return {kLive + 1, 0};
  }
  c0 = s.below_c;
  w0 = s.below_w;
  int bits_left = 15;  // key bits below the first level (keys up to 2^25 in 1024 bins of 2^15)
#pragma unroll 1
  while (bits_left) {
    const int take = bits_left == 15 ? 10 : 5;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.count[i] = 0;
      s.weight[i] = 0;
    }
    __syncthreads();
    const int shift = bits_left - take;
    for (int j = threadIdx.x; j < row.vocab; j += kThreads) {
      const uint32_t k = row.key(j);
      if (k < kLive && (k >> bits_left) == prefix) {
        const uint32_t b = (k >> shift) & ((1u << take) - 1);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.weight[b], weight_of(k));
      }
    }
    __syncthreads();
    find_bin(s, by_count, aim, c0, w0, 1 << take);
    prefix = prefix << take | s.bin;
    c0 = s.below_c;
    w0 = s.below_w;
    bits_left = shift;
  }
  const unsigned long long w = weight_of(prefix);
  const uint32_t n = s.count[prefix & 31];
  // of the n tokens with this key, the first one that reaches the aim is the last that stays
  uint32_t ties;
  if (by_count) {
    ties = (uint32_t)(aim - (double)c0);
  } else {
    ties = n;
    if (w) {
      double k = floor((aim - (double)w0) / (double)w);
      if (k < 0) k = 0;
      if (k > n) k = n;
      while (k > 0 && (double)w0 + (k - 1) * (double)w >= aim) k -= 1;
      while (k < n && (double)w0 + k * (double)w < aim) k += 1;
      ties = (uint32_t)k;
    }
  }
  kept_w = w0 + ties * w;
  return {prefix, ties};
}

template <typename T>
__device__ void first_level(Smem& s, const Row<T>& row) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.count[i] = 0;
    s.weight[i] = 0;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < row.vocab; j += kThreads) {
    const uint32_t k = row.key(j);
    if (k < kLive) {
      atomicAdd(&s.count[k >> 15], 1u);
      atomicAdd(&s.weight[k >> 15], weight_of(k));
    }
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ Smem s;
  __shared__ unsigned long long s_w[kWarps], s_c[kWarps];
  pdl_enter();
  const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Row<T> row;
  row.x = static_cast<const T*>(a.logits) + (long long)r * a.ld;
  row.vocab = a.vocab;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.vocab; j += kThreads) m = fmaxf(m, to_float(row.x[j]));
  m = block_reduce(m, s.scratchf, [](float p, float q) { return fmaxf(p, q); });
  if (m == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = __int_as_float(0x7fc00000);
    }
    return;
  }
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  row.m = m;
  row.c = temp > 0.f ? __fmul_rn(__frcp_rn(temp), 1.4426950408889634f) : INFINITY;  // 0: all but the maximum are deepest
  Cut cut = {kLive + 1, 0};
  if (!(temp > 0.f)) {
    cut = {0, 1};
  } else {
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.f;
    const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
    if (by_k || by_p) {
      first_level(s, row);
      unsigned long long kept = 0;
      Cut ck = cut;
      if (by_k) ck = find_cut(s, row, true, (double)k, kept);
      cut = ck;
      if (by_p) {
        if (by_k) first_level(s, row);
        unsigned long long total = kept;
        if (!by_k || kept == ~0ull)
          total = block_reduce(s.weight[threadIdx.x], s.scratch64,
                               [](unsigned long long x, unsigned long long y) { return x + y; });
        const double aim = (double)p * (double)total;
        Cut cp = {0, 1};
        if (aim > 0) cp = find_cut(s, row, false, aim, kept);
        if (cp.key < cut.key || (cp.key == cut.key && cp.ties < cut.ties)) cut = cp;
      }
    }
    if (cut.key == 0 && cut.ties == 0) cut.ties = 1;
  }
  const float mp = a.min_p ? a.min_p[r] : 0.f;
  const double least = mp > 0.f ? fmin((double)mp, 1.0) * 2147483648.0 : 0.0;
  // kept weight and ties of every warp's segment of the row
  const int seg = (a.vocab + kWarps * 32 - 1) / (kWarps * 32) * 32;
  const int lo = warp * seg, hi = min(a.vocab, lo + seg);
  unsigned long long w = 0;
  uint32_t n = 0;
  for (int j = lo + lane; j < hi; j += 32) {
    const uint32_t k = row.key(j);
    if (k < cut.key) {
      const unsigned long long x = weight_of(k);
      if ((double)x >= least) w += x;
    } else if (k == cut.key) {
      n += 1;
    }
  }
  for (int o = 16; o; o >>= 1) {
    w += __shfl_xor_sync(~0u, w, o);
    n += __shfl_xor_sync(~0u, n, o);
  }
  __syncthreads();
  if (lane == 0) {
    s_w[warp] = w;
    s_c[warp] = n;
  }
  __syncthreads();
  unsigned long long tie_w = weight_of(cut.key);
  if ((double)tie_w < least) tie_w = 0;
  unsigned long long total = 0, ties_left = cut.ties, mine = 0, mine_ties = 0;
  for (int i = 0; i < kWarps; ++i) {
    const unsigned long long k = s_c[i] < ties_left ? s_c[i] : ties_left;
    const unsigned long long x = s_w[i] + k * tie_w;
    if (i < warp) mine += x;
    if (i == warp) mine_ties = ties_left, w = x;
    ties_left -= k;
    total += x;
  }
  unsigned long long aim = (unsigned long long)((double)a.u[r] * (double)total);
  if (aim >= total) aim = total - 1;
  if (mine <= aim && aim < mine + w) {  // one warp: walk its segment in index order
    unsigned long long run = mine, left = mine_ties;
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      const uint32_t k = j < hi ? row.key(j) : kLive + 2;
      const uint32_t ties = __ballot_sync(~0u, k == cut.key && j < hi);
      unsigned long long x = 0;
      if (k < cut.key) {
        x = weight_of(k);
        if ((double)x < least) x = 0;
      } else if (k == cut.key && j < hi && __popc(ties & ((1u << lane) - 1)) < left) {
        x = tie_w;
      }
      unsigned long long inc = x;
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long p = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += p;
      }
      const uint32_t over = __ballot_sync(~0u, run + inc > aim);
      if (over) {
        if (lane == __ffs(over) - 1) {
          a.tokens[r] = j;
          if (a.logprobs)
            a.logprobs[r] = -(float)k * (1.f / kSteps) * 0.69314718056f - logf((float)((double)total * (1.0 / 2147483648.0)));
        }
        break;
      }
      run += __shfl_sync(~0u, inc, 31);
      const unsigned long long nt = __popc(ties);
      left -= nt < left ? nt : left;
    }
  }
}

}  // namespace
}  // namespace b2p

using namespace b2p;

extern "C" int b2p_sample(const void* logits, int ld, int rows, int vocab, int dtype, const float* u,
                          const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                          int32_t* tokens, float* logprobs, void* stream) {
  B2P_REQUIRE(rows >= 0, "rows must not be negative");
  B2P_REQUIRE(vocab >= 1 && vocab < (1 << 21), "vocab must be from 1 to 2^21 - 1 (got %d)", vocab);
  B2P_REQUIRE(dtype == B2P_F16 || dtype == B2P_BF16 || dtype == B2P_F32,
              "dtype must be B2P_F16, B2P_BF16 or B2P_F32");
  if (rows == 0) return B2P_OK;
  B2P_REQUIRE(logits && u && tokens, "null logits, u or tokens");
  B2P_REQUIRE(ld >= vocab, "ld (%d) < vocab (%d)", ld, vocab);
  DeviceCtx* c = nullptr;
  if (int rc = ctx_get(&c)) return rc;
  SampleArgs a;
  a.logits = logits;
  a.u = u;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.ld = ld;
  a.vocab = vocab;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kern = dtype == B2P_F32 ? sample_kernel<float> : dtype == B2P_F16 ? sample_kernel<__half> : sample_kernel<__nv_bfloat16>;
  B2P_CHECK_CUDA(launch_pdl(kern, dim3(rows), dim3(kThreads), 0, st, a));
  B2P_POST_LAUNCH();
  return B2P_OK;
}
