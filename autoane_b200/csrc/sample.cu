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
// sample_kernel: a CTA has a row and reads it from memory once, for the maximum,
// and then once or a few times more from the L2 cache (or L1):
//   top-k     Every thread keeps the maximum of its own tokens. The k-th largest
//             of these is no more than the k-th largest token, and little less
//             when k is small against the threads, so its bin bounds the tokens
//             to gather: a histogram of one entry a thread. They are sorted, and
//             top-p, min-p and the draw go by that list alone.
//   top-p     (without top-k) A histogram of the weights; the tokens of the bin
//             where the cut lies are gathered and sorted. The vectors that may hold
//             such a token, or a likelier one, are queued first.
//   the rest  Sums of the kept weights by warp, each with a segment of the row;
//             the warp that has the drawn sum walks through its segment.
// A list of more than 2048 tokens (many equal logits), or a queue of more vectors, is
// left for refining the histogram (long_row): six more passes over the row, a token a
// load. A nucleus comes to that where its tokens lie in more than 2048 vectors, as over a
// whole vocabulary at ordinary temperatures. Measured, normal logits of deviation 2.7,
// top-p 0.9 at T 0.7 (queued) / T 1 (long): a row of 49152 in 32 bit 32 / 125 us, 33 rows
// 35 / 133, 256 rows in 16 bit 62 / 245.
// Bound: reading the logits; in practice, for few rows the latency of the passes, for
// many that of the second one's reads from L2 at 32 warps an SM (issue 31%, the
// exponential's unit 30% busy).
// Measured: a row of 49152 (top-k 50) 10 us, 33 rows of 16893 (top-p 0.95) 25 us, 256
// rows of 49152 in 16 bit (top-k 200, top-p, min-p) 18 us, 1024 rows of 32000 in 32 bit
// (unfiltered) 60 us, 2.2 TB/s. (A row held in the registers of a cluster of CTAs, read
// once, took 17, 29, 83 and 79 us: its barriers and exchanges cost more.)
#include <cstdint>
#include <type_traits>
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
constexpr int kList = 2048;               // gathered tokens
constexpr int kTail = 256;                // threads that sort the gathered tokens and draw from them
constexpr int kAhead = 4;                 // vectors of 16 bytes that a thread loads at a time

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
  bool flat;         // cold, or a maximum or c of inf: only the largest logits weigh anything
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
__device__ __forceinline__ float key_of(float x, const Params& q) {
  if (q.flat) return x == q.m ? 0.f : INFINITY;
  return key_of(x, q.m, q.c);
}
// key >> 15, below kLive (by an addition that rounds down: conversions run at the exponential's rate)
__device__ __forceinline__ uint32_t bin_of(float key) {
  return __float_as_uint(__fadd_rz(key * (1.f / 32768.f), 8388608.f)) & 1023u;
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
  Found found;  // bin kBins before each use
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
// The first bin at which the measure (counts, or weights) reaches `aim` (> 0), into found after the next barrier; c, w:
// scan_bins' sums.
template <int NT>
__device__ __forceinline__ void find_bin(Scan<NT>& s, const uint32_t* count, const u64* weight, u64 c, u64 w,
                                         bool by_count, u64 aim) {
  constexpr int kEach = kBins / NT;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = threadIdx.x * kEach + i;
    const u64 nc = c + count[b], nw = w + weight[b];
    if (nc > c && (by_count ? c : w) < aim && (by_count ? nc : nw) >= aim) s.found = {b, c, w};  // one bin at most
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

__device__ __forceinline__ uint32_t bits_of(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t bits_of(__half x) { return __half_as_ushort(x); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t b) {
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(b);
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(__ushort_as_half((unsigned short)b));
  else
    return __uint_as_float(b << 16);
}
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// ---------------------------------------------------------------------------
// The cut by a refined histogram, for rows with more tokens near it than the list
// holds.
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
    if (threadIdx.x == 0) s.scan.found = {kBins, 0, 0};
    __syncthreads();
    find_bin<NT>(s.scan, s.count, s.weight, c + c0, w + w0, by_count, aim);
    __syncthreads();
    const Found f = s.scan.found;
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
__device__ __noinline__ void long_row(LongMem<NT>& s, SampleArgs a, int r, const T* x, Params q) {
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

// ---------------------------------------------------------------------------
// sample_kernel.
// ---------------------------------------------------------------------------
template <int NT>
struct Mem {
  union {
    struct {
      uint32_t count[kBins];
      uint32_t piece[3][kBins];  // weights, in pieces of so few bits that no sum passes 32
    } h;
    struct {
      u64 list[kList];
      int32_t queue[kList];  // vectors that may hold tokens of the list
    };
    LongMem<NT> far;
  };
  uint32_t listed, queued;
  u64 warp[NT / 32], total;
  float warp_m[NT / 32];
  int bin;
  u64 before;
  Cut cut;
};

// A barrier of the first N threads: all NT, or the tail.
template <int NT, int N>
__device__ __forceinline__ void sync_n() {
  asm volatile("bar.sync %0, %1;" ::"n"(N == NT ? 0 : 1), "n"(N) : "memory");
}

// Sum of x over the threads before this one, and over all N.
template <int NT, int N>
__device__ __forceinline__ u64 block_scan(Mem<NT>& s, u64 x, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 p = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += p;
    }
    return v;
  };
  const u64 inc = scan(x);
  sync_n<NT, N>();
  if (lane == 31) s.warp[warp] = inc;
  sync_n<NT, N>();
  if (warp == 0) {
    const u64 own = lane < N / 32 ? s.warp[lane] : 0, upto = scan(own);
    if (lane < N / 32) s.warp[lane] = upto - own;
    if (lane == 31) s.total = upto;
  }
  sync_n<NT, N>();
  total = s.total;
  return s.warp[warp] + inc - x;
}

// The first bin at which the running sum of of(bin) reaches aim (> 0), kBins if none; s.before: the sum before it.
template <int NT, typename F, typename A>
__device__ __forceinline__ int first_bin(Mem<NT>& s, u64& total, F&& of, A&& aim_of_total) {
  constexpr int kEach = kBins / NT;
  u64 v[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += v[i] = of(threadIdx.x * kEach + i);
  if (threadIdx.x == 0) s.bin = kBins;
  u64 before = block_scan<NT, NT>(s, sum, total);
  const u64 aim = aim_of_total(total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (before < aim && before + v[i] >= aim) {  // one bin at most
      s.bin = threadIdx.x * kEach + i;
      s.before = before;
    }
    before += v[i];
  }
  __syncthreads();
  return s.bin;
}

// Sorts list[0, n) upwards, by the tail's threads (bitonic); places up to the next power of two are overwritten. Strides
// below 32 go by shuffles.
template <int NT>
__device__ __forceinline__ void sort_list(u64* list, int n) {
  const int lane = threadIdx.x & 31;
  int places = 32;
  while (places < n) places *= 2;
  for (int i = n + threadIdx.x; i < places; i += kTail) list[i] = ~0ull;
  sync_n<NT, kTail>();
#pragma unroll 1
  for (int size = 32; size <= places; size *= 2) {
#pragma unroll 1
    for (int stride = size / 2; stride >= 32; stride /= 2) {
      for (int t = threadIdx.x; t < places / 2; t += kTail) {
        const int i = 2 * t - (t & (stride - 1));
        const u64 x = list[i], y = list[i + stride];
        if ((x > y) == !(i & size)) {
          list[i] = y;
          list[i + stride] = x;
        }
      }
      sync_n<NT, kTail>();
    }
    for (int i = threadIdx.x; i - lane < places; i += kTail) {
      u64 x = list[i];
      auto strides = [&](int of, int first) {
#pragma unroll
        for (int stride = first; stride; stride /= 2) {
          const u64 y = __shfl_xor_sync(~0u, x, stride);
          const bool least = !(i & stride) == !(i & of);
          x = least == (y < x) ? y : x;
        }
      };
      if (size == 32) {  // the smaller sizes first
        strides(2, 1);
        strides(4, 2);
        strides(8, 4);
        strides(16, 8);
      }
      strides(size, 16);
      list[i] = x;
    }
    sync_n<NT, kTail>();
  }
}

// A row as vectors of 16 bytes: it begins `skew` places into the first one, if it does not begin on 16 bytes.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  int skew, vocab, lo, hi;  // the warp's segment, in vectors
  __device__ __forceinline__ int index(int v) const { return v * kVec - skew; }
  // the vector whose first token is j; places outside [0, end) are -inf
  __device__ __forceinline__ uint4 load_at(int j, int end) const {
    if (j >= 0 && j + kVec <= end) return *reinterpret_cast<const uint4*>(x + j);
    uint32_t w[4] = {};
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      w[k * sizeof(T) / 4] |= (j + k >= 0 && j + k < end ? bits_of(x[j + k]) : bits_of(T(-INFINITY)))
                              << (k * sizeof(T) % 4 * 8);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // v and those 32, 64, ... further (for the warp's 32 lanes in a row)
  __device__ __forceinline__ void load(int v, uint4 (&e)[kAhead]) const {
    const int v0 = v - (int)(threadIdx.x & 31);
    if (v0 >= (skew != 0) && v0 + 32 * kAhead <= min(hi, (vocab + skew) / kVec)) {
      const uint4* p = reinterpret_cast<const uint4*>(x - skew) + v;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) e[i] = p[32 * i];
    } else {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) e[i] = load_at(index(v + 32 * i), v + 32 * i < hi ? vocab : 0);
    }
  }
  static __device__ __forceinline__ float value(const uint4& e, int k) {
    const uint32_t w = k * sizeof(T) / 4 == 0 ? e.x : k * sizeof(T) / 4 == 1 ? e.y : k * sizeof(T) / 4 == 2 ? e.z : e.w;
    return from_bits<T>(w >> (k * sizeof(T) % 4 * 8));
  }
  static __device__ __forceinline__ float most(const uint4& e) {  // the maximum of the vector
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf(value(e, 0), value(e, 1)), fmaxf(value(e, 2), value(e, 3)));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      auto two = [](uint32_t w) { return *reinterpret_cast<T2*>(&w); };
      const T2 m = __hmax2(__hmax2(two(e.x), two(e.y)), __hmax2(two(e.z), two(e.w)));
      return fmaxf(to_float(m.x), to_float(m.y));
    }
  }
  // f(index of the first, values), for the lane's vectors of the warp's segment, in order. (A long f's code is there
  // once: four copies are slower by their way through the instruction cache, as most rows run them a few times only.)
  template <bool kLong = true, typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int v = lo + lane; v - lane < hi; v += 32 * kAhead) {
      uint4 e[kAhead];
      load(v, e);
      if constexpr (kLong) {
#pragma unroll 1
        for (int i = 0; i < kAhead && v - lane + 32 * i < hi; ++i) {
          f(index(v + 32 * i), e[0]);
#pragma unroll
          for (int n = 1; n < kAhead; ++n) e[n - 1] = e[n];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f(index(v + 32 * i), e[i]);
      }
    }
  }
};

// A logit that no token of a key up to `key` is below: the key's, less what rounding may have taken from it (2^-24 of
// the difference, of the product and of m - x here, each).
__device__ __forceinline__ float least_logit(float key, const Params& q) {
  if (q.flat) return q.m;
  const float d = (key + 1.f) / q.c;
  return q.m - d - (fabsf(q.m) + d) * 0x1p-20f;
}

// Gathers the tokens of keys [from, to): the vectors that may hold some are queued, and then taken one a thread. False
// if there are more than the list or the queue holds.
template <int NT, typename T>
__device__ __forceinline__ bool gather(Mem<NT>& s, const Row<T>& row, const Params& q, float from, float to) {
  constexpr int kVec = Row<T>::kVec;
  if (threadIdx.x == 0) s.listed = s.queued = 0;
  __syncthreads();  // (the histogram is done with, too)
  // (not -inf, which it is at an infinite temperature: the vectors that a warp loads past its segment read as -inf, and
  // are real ones of the next warps)
  const float low = fmaxf(least_logit(to, q), -3.402823466e38f);
  row.template each<false>([&](int j, const uint4& e) {
    if (Row<T>::most(e) >= low) {
      const uint32_t at = atomicAdd(&s.queued, 1u);
      if (at < kList) s.queue[at] = j;
    }
  });
  __syncthreads();
  const int queued = (int)s.queued;
  if (queued > kList) return false;
#pragma unroll 1
  for (int t = threadIdx.x; t < queued; t += NT) {
    const int j = s.queue[t];
    const uint4 e = row.load_at(j, row.vocab);
    float key[kVec];
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      key[k] = key_of(Row<T>::value(e, k), q);
      mine |= (uint32_t)(key[k] >= from && key[k] < to) << k;
    }
    if (mine) {
      uint32_t at = atomicAdd(&s.listed, (uint32_t)__popc(mine));
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        if (mine >> k & 1) {
          if (at < kList) s.list[at] = token_of((uint32_t)key[k], j + k);
          ++at;
        }
      }
    }
  }
  __syncthreads();
  return s.listed <= kList;
}

// top-k's row, all of whose kept tokens are in the list, by the tail's threads.
template <int NT>
__device__ __forceinline__ void draw_from_list(Mem<NT>& s, const SampleArgs& a, int r, const Params& q, int k) {
  constexpr int kEach = kList / kTail;
  const int n = (int)s.listed, i0 = threadIdx.x * kEach;
  sort_list<NT>(s.list, n);
  u64 me[kEach], sum = 0, total;
  uint32_t w[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool in = i0 + i < n && i0 + i < k;
    me[i] = in ? s.list[i0 + i] : 0;
    w[i] = in ? weight_of((float)(uint32_t)(me[i] >> 21)) : 0;
    sum += w[i];
  }
  u64 before = block_scan<NT, kTail>(s, sum, total);
  const u64 most = q.p < 1.f ? max(p_aim(q.p, total), (u64)1) : total;
  u64 stay = 0;  // tokens: the first of the list
  sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const u64 next = before + w[i];
    if (!(before < most && w[i] >= q.least)) w[i] = 0;
    before = next;
    stay += w[i] != 0;
    sum += w[i];
  }
  block_scan<NT, kTail>(s, sum, total);
  u64 kept;
  block_scan<NT, kTail>(s, stay, kept);
  // in index order
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (w[i]) s.list[i0 + i] = (me[i] & ((1u << 21) - 1)) << 32 | me[i] >> 21;
  sync_n<NT, kTail>();
  sort_list<NT>(s.list, (int)kept);
  sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    me[i] = i0 + i < (int)kept ? s.list[i0 + i] : 0;
    w[i] = i0 + i < (int)kept ? weight_of((float)(uint32_t)me[i]) : 0;
    sum += w[i];
  }
  u64 same;
  before = block_scan<NT, kTail>(s, sum, same);
  const u64 aim = aim_of(q.u, total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (before <= aim && aim < before + w[i]) put(a, r, (int)(me[i] >> 32), (float)(uint32_t)me[i], total);
    before += w[i];
  }
}

// top-p's cut from the gathered tokens of its bin, by the tail's threads.
template <int NT>
__device__ __forceinline__ void cut_of_list(Mem<NT>& s, u64 before, u64 aim) {
  constexpr int kEach = kList / kTail;
  const int n = (int)s.listed, i0 = threadIdx.x * kEach;
  sort_list<NT>(s.list, n);
  uint32_t w[kEach];
  u64 sum = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    w[i] = i0 + i < n ? weight_of((float)(uint32_t)(s.list[i0 + i] >> 21)) : 0;
    sum += w[i];
  }
  before += block_scan<NT, kTail>(s, sum, total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (before < aim && before + w[i] >= aim) s.cut = s.list[i0 + i];  // one token
    before += w[i];
  }
}

// (64 registers, 1024 threads an SM: with 48 or 40 for 5 or 6 blocks of 256, 1024 rows of 32000 take 65 / 69 us, not 60.)
template <int NT, typename T>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(SampleArgs a) {
  constexpr int kVec = Row<T>::kVec, kWarps = NT / 32;
  __shared__ __align__(16) Mem<NT> s;
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.x;
  Row<T> row;
  row.x = static_cast<const T*>(a.logits) + (long long)r * a.ld;
  row.vocab = a.vocab;
  row.skew = (int)((reinterpret_cast<uintptr_t>(row.x) & 15u) / sizeof(T));
  const int vectors = (a.vocab + row.skew + kVec - 1) / kVec, seg = (vectors + NT - 1) / NT * 32;
  row.lo = min(vectors, warp * seg);
  row.hi = min(vectors, row.lo + seg);
  Params q = params_of(a, r);
  // the thread's and the row's maximum
  float mine = -INFINITY;
  row.template each<false>([&](int, const uint4& e) {
    mine = fmaxf(mine, Row<T>::most(e));
  });
  float m = mine;
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if (lane == 0) s.warp_m[warp] = m;
  for (int i = threadIdx.x; i < kBins; i += NT) s.h.count[i] = s.h.piece[0][i] = s.h.piece[1][i] = s.h.piece[2][i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) m = fmaxf(m, s.warp_m[i]);
  if (m == -INFINITY) {  // (or NaN alone)
    if (threadIdx.x == 0) put_none(a, r);
    return;
  }
  q.m = m;
  q.flat = q.cold || m == INFINITY || q.c == INFINITY;

  const int k = q.cold ? 1 : q.k;
  u64 total;
  if (k) {
    // a bin that holds the k-th token, or a lower one: by the threads' maxima where k is small against them (half of
    // them: 1.4 k tokens lie above it, if they are spread evenly), else by all tokens. (128 rows of 32000, k 1000, 1024
    // threads: 103 us by the maxima, as too many tokens lie above, 27 by all.)
    auto count = [&](int b) -> u64 { return s.h.count[b]; };
    auto all_of_k = [&](u64) -> u64 { return (u64)k; };
    int bin = kBins;
    if (2 * k <= NT) {
      const float key = key_of(mine, q);
      if (key < kLive) atomicAdd(&s.h.count[bin_of(key)], 1u);
      __syncthreads();
      bin = first_bin<NT>(s, total, count, all_of_k);
    }
    if (bin == kBins) {
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += NT) s.h.count[i] = 0;
      __syncthreads();
      row.each([&](int, const uint4& e) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float x = key_of(Row<T>::value(e, i), q);
          if (x < kLive) atomicAdd(&s.h.count[bin_of(x)], 1u);
        }
      });
      __syncthreads();
      bin = first_bin<NT>(s, total, count, all_of_k);
    }
    if (bin < kBins) {  // (else fewer than k tokens weigh anything)
      if (gather<NT, T>(s, row, q, 0.f, (float)((bin + 1) << 15))) {
        if (threadIdx.x < kTail) draw_from_list<NT>(s, a, r, q, k);
      } else {
        long_row<NT, T>(s.far, a, r, row.x, q);
      }
      return;
    }
  }
  Cut cut = kNoCut;
  if (q.p < 1.f) {
    // (of up to 2^16 tokens, 16 bits of each; of up to 2^21, 11)
    const int bits = a.vocab <= 1 << 16 ? 16 : 11;
    const uint32_t mask = (1u << bits) - 1;
    auto weight = [&](int b) {
      return s.h.piece[0][b] + ((u64)s.h.piece[1][b] << bits) + ((u64)s.h.piece[2][b] << 2 * bits);
    };
    auto aim_of_all = [&](u64 all) { return max(p_aim(q.p, all), (u64)1); };
    row.each([&](int, const uint4& e) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float x = key_of(Row<T>::value(e, i), q);
        if (x < kLive) {
          const uint32_t w = weight_of(x), b = bin_of(x), low = w & mask, mid = w >> bits & mask;
          if (low) atomicAdd(&s.h.piece[0][b], low);
          if (mid) atomicAdd(&s.h.piece[1][b], mid);
          if (bits < 16 && w >> 2 * bits) atomicAdd(&s.h.piece[2][b], w >> 2 * bits);
        }
      }
    });
    __syncthreads();
    const int bin = first_bin<NT>(s, total, weight, aim_of_all);
    const u64 before = s.before;
    if (!gather<NT, T>(s, row, q, (float)(bin << 15), (float)((bin + 1) << 15))) {
      long_row<NT, T>(s.far, a, r, row.x, q);
      return;
    }
    if (threadIdx.x < kTail) cut_of_list<NT>(s, before, aim_of_all(total));
    __syncthreads();
    cut = s.cut;
  }

  // kept weight of every warp and of the row
  const float cut_key = (float)(cut >> 21);
  const int cut_index = (int)(cut & ((1u << 21) - 1));
  auto kept = [&](float x, int j, float& key) -> uint32_t {  // weight of token j, 0 if it does not stay
    key = key_of(x, q);
    const uint32_t y = stays(key, j, cut_key, cut_index) ? weight_of(key) : 0;
    return y >= q.least ? y : 0;
  };
  const float low = least_logit(cut_key, q);
  u64 sum = 0;
  float key;
  if (cut == kNoCut && q.least == 0 && !q.flat)
    row.template each<false>([&](int, const uint4& e) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum += weight_of(key_of(Row<T>::value(e, i), q.m, q.c));
    });
  else
    row.each([&](int j, const uint4& e) {
      if (!(Row<T>::most(e) >= low)) return;
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum += kept(Row<T>::value(e, i), j + i, key);
    });
  u64 run = block_scan<NT, NT>(s, sum, total);
  run = __shfl_sync(~0u, run, 0);
  const u64 aim = aim_of(q.u, total);
  sum = warp_sum(sum);
  if (aim < run || aim - run >= sum) return;
  // the warp that has it: the loads, then the load, the lane and the token at which the running sum passes the aim
#pragma unroll 1
  for (int v = row.lo + lane; v - lane < row.hi; v += 32 * kAhead) {
    uint4 e[kAhead];
    u64 own[kAhead], all = 0;
    row.load(v, e);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      own[i] = 0;
#pragma unroll
      for (int n = 0; n < kVec; ++n) own[i] += kept(Row<T>::value(e[i], n), row.index(v + 32 * i) + n, key);
      all += own[i];
    }
    all = warp_sum(all);
    if (run + all <= aim) {
      run += all;
      continue;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      u64 inc = own[i];
      for (int o = 1; o < 32; o <<= 1) {
        const u64 p = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += p;
      }
      const uint32_t over = __ballot_sync(~0u, run + inc > aim);
      if (over) {
        if (lane == __ffs(over) - 1) {
          run += inc - own[i];
#pragma unroll
          for (int n = 0; n < kVec; ++n) {
            const int j = row.index(v + 32 * i) + n;
            const uint32_t y = kept(Row<T>::value(e[i], n), j, key);
            if (run <= aim && aim < run + y) put(a, r, j, key, total);
            run += y;
          }
        }
        return;
      }
      run += __shfl_sync(~0u, inc, 31);
    }
  }
}

template <typename T>
int launch_t(const SampleArgs& a, int rows, const DeviceCtx* c, cudaStream_t st) {
  // As many threads for a row as leave all rows resident at once. Measured with 1024 / 512 / 256 threads: 64 rows of
  // 49152 (top-k 200) 14 / 15 / 34 us, 148 of 32000 (unfiltered) 13 / 17 / 26; 256 of 49152 29 / 20 / 49, 296 of 32000
  // 24 / 22 / 30; 1024 of 49152 (top-k 50) 85 / 50 / 40, 4096 of 2000 238 / 130 / 77.
  const int sms = c->num_sms;
  const int nt = rows <= sms ? 1024 : rows <= 2 * sms ? 512 : 256;
  if (nt == 1024)
    B2P_CHECK_CUDA(launch_pdl(sample_kernel<1024, T>, dim3(rows), dim3(1024), 0, st, a));
  else if (nt == 512)
    B2P_CHECK_CUDA(launch_pdl(sample_kernel<512, T>, dim3(rows), dim3(512), 0, st, a));
  else
    B2P_CHECK_CUDA(launch_pdl(sample_kernel<256, T>, dim3(rows), dim3(256), 0, st, a));
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
