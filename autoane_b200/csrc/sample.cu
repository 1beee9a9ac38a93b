// sample.cu — sampling a token per row of logits with temperature, top-k, top-p
// and min-p, from given uniform numbers.
//
// A token's weight is an integer, w = round(2^31 · 2^-depth), its depth below
// the row's maximum taken in steps of 2^-20 (the key, at most 2^26), so every sum
// is exact in 64 bits whatever its order: the filters and the draw are the same in
// every run. The kept tokens are a prefix of the ranking by (key, index), so each
// filter is a cut: the last of them. top-k's cut is found by counts, top-p's by
// weights, both in a histogram of the upper key bits (1024 bins of 1/32 octave);
// the tokens of the bins where the cuts lie are then gathered and ranked.
//
// sample_kernel: a cluster of up to 8 CTAs has a row, 8192 logits a CTA, 32 in
// the registers of each thread, so that a row is read once. The CTAs exchange
// maxima, histograms and sums through each other's shared memory; the first one
// decides. Four CTAs of an SM, mostly of different rows, cover each other's loads
// and exchanges. Bound: reading the logits; in practice the exponential and the
// two conversions of each token (16 a cycle and SM), and the exchanges' latency.
//
// sample_long_kernel: a row of more than 65536 logits by one CTA that reads it
// several times (the same steps, the histogram refined by further passes). It is
// also how a row of sample_kernel ends whose cut lies among more than 2048 tokens
// of one bin (many equal logits).
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "engine.cuh"
#include "ptx.cuh"

namespace b2p {
namespace {

typedef unsigned long long u64;

constexpr float kSteps = 1048576.f;       // key steps per unit of depth
constexpr float kLive = 32.f * kSteps;    // keys from here on weigh nothing: 2^31 · 2^-32 rounds to 0
constexpr float kOne = 2147483648.f;      // the weight of key 0
constexpr int kBins = 1024;               // of the histogram: 2^15 keys each
constexpr int kThreads = 256;             // sample_kernel
constexpr int kWarps = kThreads / 32;
constexpr int kPer = 32;                  // logits of a thread
constexpr int kSlice = kThreads * kPer;
constexpr int kMaxCtas = 8;
constexpr int kList = 2048;               // gathered tokens
constexpr int kLongThreads = 1024;        // sample_long_kernel

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

// A row's parameters, as every thread reads them.
struct Params {
  float m, c;        // the maximum; log2(e) / T · kSteps
  bool cold;         // T <= 0: the first of the largest logits
  int k;             // 0: off
  float p;           // 1: off
  uint32_t least;    // min-p as a weight
  float u;
};

// (all but the maximum, which is not known yet when they are read)
__device__ __forceinline__ Params params_of(const SampleArgs& a, int r) {
  Params q;
  const float t = a.temperature ? a.temperature[r] : 1.f;
  q.m = 0.f;
  q.u = a.u[r];
  q.cold = !(t > 0.f);
  q.c = q.cold ? 0.f : __fmul_rn(__frcp_rn(t), 1.4426950408889634f) * kSteps;
  const int k = a.top_k ? a.top_k[r] : 0;
  q.k = k > 0 && k < a.vocab ? k : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  q.p = p < 1.f ? p : 1.f;
  const float mp = a.min_p ? a.min_p[r] : 0.f;
  q.least = mp > 0.f ? (uint32_t)ceil(fmin((double)mp, 1.0) * 2147483648.0) : 0u;
  return q;
}

// The key of logit x, an integer held in a float (exactly: above 2^23 the product is one already). A NaN logit's is
// NaN, which no comparison below takes in and whose weight is 0; that of -inf is inf, whose weight is 0 too.
__device__ __forceinline__ float key_of(float x, float m, float c) {
  const float d = (m - x) * c;
  return d < 8388608.f ? __fadd_rn(__fadd_rn(d, 8388608.f), -8388608.f) : d;
}
// The same in rows that are cold, or whose maximum is inf: only the largest logits count.
__device__ __forceinline__ float key_of(float x, const Params& q) {
  if (q.cold || q.m == INFINITY) return x == q.m ? 0.f : INFINITY;
  return key_of(x, q.m, q.c);
}
__device__ __forceinline__ uint32_t weight_of(float key) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(key * (-1.f / kSteps)));
  return __float2uint_rn(e * kOne);
}

// The last token that stays, as key << 21 | index. No token: kNoCut, the largest live one.
typedef u64 Cut;
constexpr Cut kNoCut = ((u64)kLive << 21) - 1;
__device__ __forceinline__ Cut token_of(uint32_t key, int index) { return (u64)key << 21 | (u64)index; }
__device__ __forceinline__ bool stays(float key, int index, float cut_key, int cut_index) {
  return key < cut_key || (key == cut_key && index <= cut_index);
}

struct Found {  // a bin, and the sums before it
  int bin;
  u64 count, weight;
};

template <int NT>
struct Scan {
  u64 c[NT / 32], w[NT / 32];
  Found found[3];  // bin kBins before each use
};

// A histogram's running sums: each thread has those before its kBins / NT bins.
template <int NT>
__device__ __forceinline__ void scan_bins(Scan<NT>& s, const uint32_t* count, const u64* weight, u64& c, u64& w) {
  constexpr int kEach = kBins / NT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i0 = threadIdx.x * kEach;
  c = w = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    c += count[i0 + i];
    w += weight[i0 + i];
  }
  const u64 own_c = c, own_w = w;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 pc = __shfl_up_sync(~0u, c, o), pw = __shfl_up_sync(~0u, w, o);
    if (lane >= o) {
      c += pc;
      w += pw;
    }
  }
  if (lane == 31) {
    s.c[warp] = c;
    s.w[warp] = w;
  }
  __syncthreads();
  c -= own_c;
  w -= own_w;
  for (int k = 0; k < warp; ++k) {
    c += s.c[k];
    w += s.w[k];
  }
}
// The first bin at which the measure (counts, or weights) reaches `aim` (> 0), into found[slot] after the next barrier;
// c, w: scan_bins' sums.
template <int NT>
__device__ __forceinline__ void find_bin(Scan<NT>& s, const uint32_t* count, const u64* weight, u64 c, u64 w,
                                         bool by_count, u64 aim, int slot) {
  constexpr int kEach = kBins / NT;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = threadIdx.x * kEach + i;
    const u64 nc = c + count[b], nw = w + weight[b];
    if (nc > c && (by_count ? c : w) < aim && (by_count ? nc : nw) >= aim) s.found[slot] = {b, c, w};  // one bin at most
    c = nc;
    w = nw;
  }
}

// top-p's aim as an integer: sums below it are below p of `kept`.
__device__ __forceinline__ u64 p_aim(float p, u64 kept) { return (u64)ceil((double)p * (double)kept); }

__device__ __forceinline__ u64 warp_sum(u64 x) {
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}
__device__ __forceinline__ u64 aim_of(float u, u64 total) {
  const u64 aim = (u64)((double)u * (double)total);
  return aim < total ? aim : total - 1;
}
__device__ __forceinline__ void put(const SampleArgs& a, int r, int token, float key, u64 total) {
  a.tokens[r] = token;
  if (a.logprobs)
    a.logprobs[r] = -key * (1.f / kSteps) * 0.69314718056f - logf((float)((double)total * (1.0 / 2147483648.0)));
}
__device__ __forceinline__ void put_none(const SampleArgs& a, int r) {
  a.tokens[r] = -1;
  if (a.logprobs) a.logprobs[r] = __int_as_float(0x7fc00000);
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// ---------------------------------------------------------------------------
// One CTA for a row in global memory.
// ---------------------------------------------------------------------------
template <int NT>
struct LongMem {
  uint32_t count[kBins];
  u64 weight[kBins];
  Scan<NT> scan;
  u64 n[NT / 32];
  int index;
};

// Histogram of the keys k with (k >> above) == prefix by their `take` next bits.
template <int NT, typename T>
__device__ void long_histogram(LongMem<NT>& s, const T* x, int vocab, const Params& q, uint32_t prefix, int above,
                               int take) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += NT) {
    s.count[i] = 0;
    s.weight[i] = 0;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < vocab; j += NT) {
    const float key = key_of(to_float(x[j]), q);
    const uint32_t k = key < kLive ? (uint32_t)key : 0;
    if (key < kLive && (k >> above) == prefix) {
      const uint32_t b = (k >> (above - take)) & ((1u << take) - 1);
      atomicAdd(&s.count[b], 1u);
      atomicAdd(&s.weight[b], (u64)weight_of(key));
    }
  }
  __syncthreads();
}

// The cut at which the measure reaches `aim` (> 0), and the weight of what it keeps; all live tokens if it never does.
template <int NT, typename T>
__device__ Cut long_cut(LongMem<NT>& s, const T* x, int vocab, const Params& q, bool by_count, u64 aim, u64& kept) {
  uint32_t prefix = 0;
  u64 c0 = 0, w0 = 0;
#pragma unroll 1
  for (int above = 25; above; above = above == 25 ? 15 : above == 15 ? 5 : 0) {
    long_histogram<NT, T>(s, x, vocab, q, prefix, above, above == 5 ? 5 : 10);
    u64 c, w;
    scan_bins<NT>(s.scan, s.count, s.weight, c, w);
    if (threadIdx.x == 0) s.scan.found[0] = {kBins, 0, 0};
    __syncthreads();
    find_bin<NT>(s.scan, s.count, s.weight, c + c0, w + w0, by_count, aim, 0);
    __syncthreads();
    const Found f = s.scan.found[0];
    if (f.bin == kBins) {  // (on the first level only)
      kept = 0;
      for (int i = 0; i < NT / 32; ++i) kept += s.scan.w[i];
      return kNoCut;
    }
    prefix = prefix << (above == 5 ? 5 : 10) | (uint32_t)f.bin;
    c0 = f.count;
    w0 = f.weight;
  }
  // of the n tokens with this key, the first that reaches the aim is the last that stays
  const uint32_t w = weight_of((float)prefix), n = s.count[prefix & 31];
  u64 ties = by_count ? aim - c0 : w ? (aim - w0 + w - 1) / w : n;
  if (ties > n) ties = n;
  kept = w0 + ties * w;
  // its index: that of the tie of this number
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seg = (vocab + NT - 1) / NT * 32;
  const int lo = min(vocab, warp * seg), hi = min(vocab, lo + seg);
  u64 mine = 0;
  for (int j = lo + lane; j < hi; j += 32) mine += key_of(to_float(x[j]), q) == (float)prefix;
  mine = warp_sum(mine);
  __syncthreads();
  if (lane == 0) s.n[warp] = mine;
  __syncthreads();
  u64 before = 0;
  for (int i = 0; i < warp; ++i) before += s.n[i];
  if (before < ties && ties <= before + mine) {
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      const uint32_t tie = __ballot_sync(~0u, j < hi && key_of(to_float(x[j]), q) == (float)prefix);
      if (before + __popc(tie) >= ties) {
        if ((tie >> lane & 1) && before + __popc(tie & ((1u << lane) - 1)) + 1 == ties) s.index = j;
        break;
      }
      before += __popc(tie);
    }
  }
  __syncthreads();
  return token_of(prefix, s.index);
}

// One warp walks [lo, hi) in index order from the sum `run` on: the first token whose running sum passes `aim`.
template <typename T>
__device__ void walk(const SampleArgs& a, int r, const T* x, const Params& q, int lo, int hi, Cut cut, u64 run, u64 aim,
                     u64 total) {
  const int lane = threadIdx.x & 31;
  const float cut_key = (float)(cut >> 21);
  const int cut_index = (int)(cut & ((1u << 21) - 1));
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int j = j0 + lane;
    const float key = j >= 0 && j < hi ? key_of(to_float(x[j]), q) : INFINITY;
    u64 y = 0;
    if (stays(key, j, cut_key, cut_index)) {
      y = weight_of(key);
      if (y < q.least) y = 0;
    }
    for (int o = 1; o < 32; o <<= 1) {
      const u64 p = __shfl_up_sync(~0u, y, o);
      if (lane >= o) y += p;
    }
    const uint32_t over = __ballot_sync(~0u, run + y > aim);
    if (over) {
      if (lane == __ffs(over) - 1) put(a, r, j, key, total);
      return;
    }
    run += __shfl_sync(~0u, y, 31);
  }
}

template <int NT, typename T>
__device__ __noinline__ void long_row(LongMem<NT>& s, const SampleArgs& a, int r, const T* x, const Params& q) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Cut cut = kNoCut;
  if (q.cold || q.k || q.p < 1.f) {
    u64 kept = 0;
    cut = long_cut<NT, T>(s, x, a.vocab, q, true, q.cold ? 1 : q.k ? (u64)q.k : ~0ull, kept);
    if (!q.cold && q.p < 1.f) {
      const Cut c = long_cut<NT, T>(s, x, a.vocab, q, false, max(p_aim(q.p, kept), (u64)1), kept);
      cut = c < cut ? c : cut;
    }
  }
  const float cut_key = (float)(cut >> 21);
  const int cut_index = (int)(cut & ((1u << 21) - 1));
  // kept weight of every warp's segment of the row
  const int seg = (a.vocab + NT - 1) / NT * 32;
  const int lo = min(a.vocab, warp * seg), hi = min(a.vocab, lo + seg);
  u64 w = 0;
  for (int j = lo + lane; j < hi; j += 32) {
    const float key = key_of(to_float(x[j]), q);
    if (stays(key, j, cut_key, cut_index)) {
      const uint32_t y = weight_of(key);
      if (y >= q.least) w += y;
    }
  }
  w = warp_sum(w);
  __syncthreads();
  if (lane == 0) s.n[warp] = w;
  __syncthreads();
  u64 total = 0, run = 0;
  for (int i = 0; i < NT / 32; ++i) {
    if (i == warp) run = total;
    total += s.n[i];
  }
  const u64 aim = aim_of(q.u, total);
  if (run <= aim && aim < run + w) walk(a, r, x, q, lo, hi, cut, run, aim, total);
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) sample_long_kernel(SampleArgs a) {
  __shared__ LongMem<kLongThreads> s;
  __shared__ float s_m[kLongThreads / 32];
  pdl_enter();
  const int r = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + (long long)r * a.ld;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.vocab; j += kLongThreads) m = fmaxf(m, to_float(x[j]));
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < kLongThreads / 32; ++i) m = fmaxf(m, s_m[i]);
  if (m == -INFINITY) {
    if (threadIdx.x == 0) put_none(a, r);
    return;
  }
  Params q = params_of(a, r);
  q.m = m;
  long_row<kLongThreads, T>(s, a, r, x, q);
}

// ---------------------------------------------------------------------------
// A cluster for a row, its logits in registers.
// ---------------------------------------------------------------------------
struct Histograms {
  // this CTA's histogram; a bin's weight in 16-bit halves (of at most 8192 tokens, so neither sum passes 32 bits)
  uint32_t count[kBins], high[kBins], low[kBins];
  // first CTA: the row's
  uint32_t all_count[kBins];
  u64 all_weight[kBins];
};
struct Ranks {  // first CTA, when the histograms have been used: of the gathered tokens
  u64 w_before[kList];
  uint32_t rank[kList];
};
struct Mem {
  union {
    Histograms h;
    Ranks g;
  };
  // first CTA: the gathered tokens and their weights
  u64 list[kList];
  uint32_t list_w[kList];
  uint32_t listed;
  Scan<kThreads> scan;
  // exchanged: by rank
  float m[kMaxCtas];
  u64 w[kMaxCtas];
  // decided by the first CTA
  int lo_bin, hi_bin, k_bin;  // gather the tokens of bins lo..hi, and of k_bin
  Cut cut;
  int long_way;
  // of the warps
  float warp_m[kWarps];
  u64 warp_w[kWarps], warp_c[kWarps];
};

template <typename V>
__device__ __forceinline__ V* remote(V* p, uint32_t rank) {  // the same variable of another CTA of the cluster
  uint64_t g;
  asm("mapa.u64 %0, %1, %2;" : "=l"(g) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<V*>(g);
}

// Over the CTA: the sum of x and the maximum of y.
__device__ __forceinline__ void block_sum_max(Mem& s, u64& x, u64& y) {
  x = warp_sum(x);
  for (int o = 16; o; o >>= 1) {
    const u64 z = __shfl_xor_sync(~0u, y, o);
    y = z > y ? z : y;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    s.warp_w[threadIdx.x >> 5] = x;
    s.warp_c[threadIdx.x >> 5] = y;
  }
  __syncthreads();
  x = y = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    x += s.warp_w[i];
    y = s.warp_c[i] > y ? s.warp_c[i] : y;
  }
}

// The row's cut, from the gathered tokens (whole bins) and the sums before top-k's and top-p's bins: the first CTA, all
// its threads. Every token's rank and the weight before it come by comparing it with every other one.
__device__ __forceinline__ Cut list_cut(Mem& s, int k, float p, const Found& fk, const Found& fp, u64 all_w) {
  const uint32_t n = s.listed;
  u64 earlier_bins = 0;  // gathered tokens of bins before top-k's
  __syncthreads();       // (every thread has its histogram figures)
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const u64 me = s.list[i];
    uint32_t rank = 0;
    u64 before = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) {
      const bool ahead = s.list[j] < me;
      rank += ahead;
      before += ahead ? s.list_w[j] : 0u;
    }
    s.g.rank[i] = rank;
    s.g.w_before[i] = before;
    earlier_bins += (int)(me >> 36) < fk.bin;
  }
  Cut cut = kNoCut;
  u64 kept = all_w, last = 0;
  if (fk.bin < kBins) {
    block_sum_max(s, earlier_bins, last);
    kept = last = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const u64 me = s.list[i];
      if ((int)(me >> 36) == fk.bin && fk.count + s.g.rank[i] - earlier_bins < (u64)k) {
        kept += s.list_w[i];
        last = me > last ? me : last;
      }
    }
    block_sum_max(s, kept, last);
    kept += fk.weight;
    cut = last;
  }
  if (p < 1.f) {
    const u64 aim = max(p_aim(p, kept), (u64)1);
    last = kept = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const u64 me = s.list[i];
      const int b = (int)(me >> 36);
      if (b >= s.lo_bin && b <= s.hi_bin && fp.weight + s.g.w_before[i] < aim) last = me > last ? me : last;
    }
    block_sum_max(s, kept, last);
    cut = last < cut ? last : cut;
  }
  return cut;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(SampleArgs a, int ctas) {
  constexpr int kVec = 16 / sizeof(T), kLoads = kPer / kVec;
  extern __shared__ __align__(16) uint8_t smem[];
  Mem& s = *reinterpret_cast<Mem*>(smem);
  // (no CTA writes to another one before that has started: the barrier's other half comes before the first write)
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = ctas > 1 ? cluster_ctarank() : 0;
  const int r = blockIdx.x / ctas;
  const T* row = static_cast<const T*>(a.logits) + (long long)r * a.ld;
  Params q = params_of(a, r);
  // A CTA's slice goes by 16-byte vectors, so the row begins `skew` places into the first one. Index order is that of
  // (rank, warp, load, lane, place in the vector).
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int first = (int)rank * kSlice + warp * (32 * kPer) + lane * kVec - skew;
  float x[kPer];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int j = first + i * 32 * kVec;
    if (j >= 0 && j + kVec <= a.vocab) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + j));
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int k = 0; k < kVec; ++k) x[i * kVec + k] = to_float(e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k) x[i * kVec + k] = j + k >= 0 && j + k < a.vocab ? to_float(row[j + k]) : -INFINITY;
    }
  }
  if (threadIdx.x < 3) s.scan.found[threadIdx.x] = {kBins, 0, 0};
  if (threadIdx.x == 0) s.listed = 0;
  // the row's maximum
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) m = fmaxf(m, x[i]);
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (lane == 0) s.warp_m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) m = fmaxf(m, s.warp_m[i]);
  if (ctas > 1) {
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (threadIdx.x < ctas) *remote(&s.m[rank], threadIdx.x) = m;
    cluster_sync();
    for (int i = 0; i < ctas; ++i) m = fmaxf(m, s.m[i]);
  }
  if (m == -INFINITY || isnan(m)) {  // (every CTA of the row; a maximum over NaN alone is a NaN)
    if (rank == 0 && threadIdx.x == 0) put_none(a, r);
    return;
  }
  q.m = m;
  if (q.cold || m == INFINITY) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = x[i] == m ? 0.f : INFINITY;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = key_of(x[i], q.m, q.c);
  }

  Cut cut = kNoCut;
  if (q.cold || q.k || q.p < 1.f) {
    const bool by_p = !q.cold && q.p < 1.f;
    const int k = q.cold ? 1 : q.k;
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.h.count[i] = s.h.high[i] = s.h.low[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (x[i] < kLive) {
        const uint32_t b = (uint32_t)x[i] >> 15;
        atomicAdd(&s.h.count[b], 1u);
        if (by_p) {
          const uint32_t w = weight_of(x[i]);
          atomicAdd(&s.h.high[b], w >> 16);
          atomicAdd(&s.h.low[b], w & 0xffffu);
        }
      }
    }
    auto sync = [&]() {
      if (ctas > 1)
        cluster_sync();
      else
        __syncthreads();
    };
    sync();
    // the row's histogram: each CTA sums some bins over the cluster, into the first one's memory
    const int each = (kBins + ctas - 1) / ctas;
    for (int b = (int)rank * each + threadIdx.x; b < min(kBins, (int)(rank + 1) * each); b += kThreads) {
      uint32_t c = 0;
      u64 w = 0;
#pragma unroll 4
      for (int i = 0; i < ctas; ++i) {
        c += *remote(&s.h.count[b], i);
        if (by_p) w += ((u64) * remote(&s.h.high[b], i) << 16) + *remote(&s.h.low[b], i);
      }
      *remote(&s.h.all_count[b], 0) = c;
      *remote(&s.h.all_weight[b], 0) = w;
    }
    sync();
    // the first CTA: where the cuts lie. top-p's aim goes by what top-k keeps, known to within top-k's bin, so a few
    // bins may hold it.
    Found fk = {kBins, 0, 0}, fp = {kBins, 0, 0};
    u64 all_w = 0;
    if (rank == 0) {
      u64 c, w;
      scan_bins<kThreads>(s.scan, s.h.all_count, s.h.all_weight, c, w);
      if (k) {
        find_bin<kThreads>(s.scan, s.h.all_count, s.h.all_weight, c, w, true, (u64)k, 0);
        __syncthreads();
        fk = s.scan.found[0];
      }
      int lo = kBins, hi = -1;
      if (by_p) {
        for (int i = 0; i < kWarps; ++i) all_w += s.scan.w[i];
        const u64 least_w = fk.bin < kBins ? fk.weight : all_w;
        const u64 most_w = fk.bin < kBins ? fk.weight + s.h.all_weight[fk.bin] : all_w;
        const u64 lo_aim = max(p_aim(q.p, least_w), (u64)1), hi_aim = max(p_aim(q.p, most_w), (u64)1);
        find_bin<kThreads>(s.scan, s.h.all_count, s.h.all_weight, c, w, false, lo_aim, 1);
        find_bin<kThreads>(s.scan, s.h.all_count, s.h.all_weight, c, w, false, hi_aim, 2);
        __syncthreads();
        fp = s.scan.found[1];
        lo = fp.bin;
        hi = s.scan.found[2].bin;
      }
      if (threadIdx.x < ctas) {
        *remote(&s.lo_bin, threadIdx.x) = lo;
        *remote(&s.hi_bin, threadIdx.x) = hi;
        *remote(&s.k_bin, threadIdx.x) = fk.bin;
      }
    }
    sync();
    if (s.k_bin < kBins || s.lo_bin < kBins) {
      // (keys up to kLive only: a bin that is none begins there)
      const float lo_key = (float)(s.lo_bin << 15), hi_key = (float)((s.hi_bin + 1) << 15);
      const float k_lo = (float)(s.k_bin << 15), k_hi = s.k_bin < kBins ? (float)((s.k_bin + 1) << 15) : k_lo;
      uint32_t* const listed = remote(&s.listed, 0);
      u64* const list = remote(&s.list[0], 0);
      uint32_t* const list_w = remote(&s.list_w[0], 0);
      // (one atomic of each warp on the first CTA's count: a round trip takes about a thousand cycles)
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        mine |= (uint32_t)((x[i] >= lo_key && x[i] < hi_key) || (x[i] >= k_lo && x[i] < k_hi)) << i;
      const uint32_t n = __popc(mine);
      uint32_t at = n;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t p = __shfl_up_sync(~0u, at, o);
        if (lane >= o) at += p;
      }
      uint32_t from = 0;
      if (lane == 31 && at) from = atomicAdd(listed, at);
      at += __shfl_sync(~0u, from, 31) - n;
      if (__any_sync(~0u, n != 0)) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (mine >> i & 1) {
            if (at < kList) {
              list[at] = token_of((uint32_t)x[i], first + (i / kVec) * 32 * kVec + i % kVec);
              list_w[at] = weight_of(x[i]);
            }
            at += 1;
          }
        }
      }
      sync();
      if (rank == 0) {
        const bool too_many = s.listed > kList;
        if (!too_many) cut = list_cut(s, k, by_p ? q.p : 1.f, fk, fp, all_w);
        if (threadIdx.x < ctas) {
          *remote(&s.cut, threadIdx.x) = cut;
          *remote(&s.long_way, threadIdx.x) = too_many;
        }
      }
      sync();
      cut = s.cut;
      if (s.long_way) {
        if (rank == 0) long_row<kThreads, T>(*reinterpret_cast<LongMem<kThreads>*>(smem), a, r, row, q);
        return;
      }
    }
  }

  // kept weight of every warp, CTA and the row
  const float cut_key = (float)(cut >> 21);
  const int cut_index = (int)(cut & ((1u << 21) - 1));
  auto kept = [&](int i) -> uint32_t {  // weight of the thread's token i, 0 if it does not stay
    const uint32_t y = stays(x[i], first + (i / kVec) * 32 * kVec + i % kVec, cut_key, cut_index) ? weight_of(x[i]) : 0;
    return y >= q.least ? y : 0;
  };
  u64 w = 0;
  if (cut == kNoCut && q.least == 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) w += weight_of(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) {  // (most loads of a row that is cut hold no token that stays)
      float least_key = x[i];
#pragma unroll
      for (int k = 1; k < kVec; ++k) least_key = fminf(least_key, x[i + k]);
      if (__any_sync(~0u, least_key <= cut_key)) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) w += kept(i + k);
      }
    }
  }
  w = warp_sum(w);
  __syncthreads();
  if (lane == 0) s.warp_w[warp] = w;
  __syncthreads();
  u64 total = 0, run = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i == warp) run = total;
    total += s.warp_w[i];
  }
  if (ctas > 1) {
    if (threadIdx.x < ctas) *remote(&s.w[rank], threadIdx.x) = total;
    cluster_sync();
    total = 0;
    for (int i = 0; i < ctas; ++i) {
      if (i == (int)rank) run += total;
      total += s.w[i];
    }
  }
  const u64 aim = aim_of(q.u, total);
  if (aim < run || aim >= run + w) return;
  // the warp that has it: the load, then the lane, then the token at which the running sum passes the aim
  uint32_t y[kVec];
  float key[kVec];
  int j = 0;
  bool here = false;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    u64 sum = 0;
#pragma unroll
    for (int k = 0; k < kVec; ++k) sum += kept(i * kVec + k);
    sum = warp_sum(sum);
    if (!here) {
      if (run + sum > aim) {
        here = true;
        j = first + i * 32 * kVec;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          y[k] = kept(i * kVec + k);
          key[k] = x[i * kVec + k];
        }
      } else {
        run += sum;
      }
    }
  }
  u64 sum = 0;
#pragma unroll
  for (int k = 0; k < kVec; ++k) sum += y[k];
  u64 inc = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 p = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += p;
  }
  const uint32_t over = __ballot_sync(~0u, run + inc > aim);
  if (lane != __ffs(over) - 1) return;
  run += inc - sum;
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    run += y[k];
    if (run > aim) {
      put(a, r, j + k, key[k], total);
      return;
    }
  }
}

template <typename T>
int launch_t(const SampleArgs& a, int rows, const DeviceCtx* c, cudaStream_t st) {
  // (a row that does not begin on 16 bytes takes part of one more vector)
  const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld * sizeof(T) % 16 == 0;
  const int ctas = (a.vocab + (aligned ? 0 : (int)(16 / sizeof(T)) - 1) + kSlice - 1) / kSlice;
  if (ctas > kMaxCtas) {
    B2P_CHECK_CUDA(launch_pdl(sample_long_kernel<T>, dim3(rows), dim3(kLongThreads), 0, st, a));
    B2P_POST_LAUNCH();
    return B2P_OK;
  }
  static_assert(sizeof(LongMem<kThreads>) <= sizeof(Mem), "the long way fits the same memory");
  static thread_local uint64_t attr_mask = 0;  // one per instantiation
  if (!(attr_mask & (1ull << (c->device & 63)))) {
    B2P_CHECK_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Mem)));
    attr_mask |= 1ull << (c->device & 63);
  }
  B2P_REQUIRE((long long)rows * ctas < (1ll << 31), "too many rows in one call");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Mem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  B2P_CHECK_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, ctas));
  B2P_POST_LAUNCH();
  return B2P_OK;
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
  B2P_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == B2P_F32 ? 4 : 2) == 0, "logits must be aligned");
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
  if (dtype == B2P_F32) return launch_t<float>(a, rows, c, st);
  return dtype == B2P_F16 ? launch_t<__half>(a, rows, c, st) : launch_t<__nv_bfloat16>(a, rows, c, st);
}
