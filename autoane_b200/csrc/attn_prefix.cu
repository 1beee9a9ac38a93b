// attn_prefix.cu — attention of a batch that shares a long prefix, over a paged
// cache of 16-bit or 8-bit keys and values.
//
// With s_j = q·k_j / 8 and any split of a row's keys into parts, each part's
//   m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j
// join to out = sum e^(m_p - M) o_p / sum e^(m_p - M) l_p, M = max m_p, and the
// log-sum-exp M + log(sum e^(m_p - M) l_p). The shared prefix is one part list
// for the rows of all sequences at once (its keys are read once for the batch);
// each sequence's suffix is another. A long prefix goes to attn_prefix_tc.cu.
// attn_join_kernel joins the parts. (Joining where a row's last part is written,
// behind a fence and a counter, took longer: 8 sequences of one query, 15 heads,
// 1024 shared keys 13.3 us in place of 8.6, 16 over 4096 34 in place of 17.)
//
// attn_rows_kernel: each warp holds 16 or 32 query rows of one KV head and runs
// over 32 keys at a time with mma.sync. Its keys and values come as they are
// stored into a ring of its own in shared memory (cp.async, up to 128 keys ahead,
// no barrier between warps) and from there into fragments: a head's 64 channels
// are taken in the order that gives each thread 16 consecutive ones of a key
// (S = Q·Kᵀ sums over channels, so Q is read in the same order) and 8 consecutive
// ones of a value (each is a column of O of its own).
//
// 8-bit caches: codes widen to 16 bit exactly. A key's scale multiplies its
// column of S in fp32. A value's scale y_j joins the exponent,
//   w_j = exp2(s_j log2e + log2 y_j - M), M near the largest of the sums so far,
// so that o = sum w_j code_j, l = sum w_j / y_j and out = o / l: the one rounding
// to 16 bit is that of w_j, as without scales, for values down to 2^-73.
//
// The weights are rounded to the compute dtype, here and in attn_prefix_tc.cu: the
// tensor cores take 16-bit pairs, and weights in two parts would double the second
// product. l is summed before the rounding. Beside the output's own rounding this makes
// the error against 64 bits 0.0023 (bf16) or 0.00030 (fp16) of the output's size, with
// weights in 32 bits 0.0017 and 0.00021.
//
// Bound: for few rows the latency of a unit's loads and of the join; for many the
// instructions around 16 x 8 tiles that hold 3 rows of 16 (group 3). 256 suffixes
// of up to 512 int8 keys, 5 KV heads: 23 us beside 7 us of reading; 8 sequences
// over 1023 + 129 keys: 9 us with the join.
#include <cstdint>
#include <type_traits>
#include "attn_prefix.cuh"
#include "ptx.cuh"

namespace b2p {
namespace {

constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kStep = 32;            // keys of one warp step
constexpr int kPitch = kKvHeadDim + 4;  // floats of a row of O in shared memory
constexpr int kMaxChunk = 4096;      // keys of one part
constexpr int kMaxChunkPages = kMaxChunk / 8 + 1;
constexpr float kSlack = 8.f;        // weights go up to 2^8 before a row's reference moves
constexpr int kMinPart = 128;        // no part shorter: its join would cost what it saves
constexpr int kSinglePages = 32;     // of a single warp's unit: a lane's each
constexpr int kWant = kSms * 4;      // blocks wanted of each list
// The prefix goes to the tcgen05 kernel from this length on, or from so many rows times keys (8-bit or 16-bit cache; the
// first pay for widening). Measured, 5 KV heads, attn_rows_kernel / tcgen05: int8, 1024 keys, 96 rows 10.7 / 12.2 us,
// 192 rows 14.2 / 13.3; 4096 keys, 24 rows 12.6 / 13.8, 48 rows 16.7 / 14.3; 8192 keys, 6 rows 16.9 / 14.5; 32768 keys,
// 96 rows 40 / 28, 768 rows 175 / 74. 16-bit, 1024 keys, 24 rows 8.6 / 8.8, 48 rows 9.5 / 9.1; 4096 keys, 6 rows
// 10.9 / 10.9, 24 rows 12.7 / 11.2.
constexpr int kTcKeys = 8192;
constexpr long long kTcWork8 = 128 * 1024, kTcWork16 = 48 * 1024;

__device__ __forceinline__ float rcp_sfu(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_sfu(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A step's keys in shared memory: K rows, V rows (16-byte chunks of a row exchanged so that the fragments' reads meet
// no bank conflict), and for 8-bit kinds the scales of 32 keys and 32 values.
template <int KIND>
struct StepMem {
  static constexpr bool kQ8 = KIND != B2P_KV_16;
  static constexpr int kRow = kQ8 ? 64 : 128;        // bytes of a key
  static constexpr int kChunks = kRow / 16;
  static constexpr int kV = kStep * kRow;            // offset of V, then of the scales
  static constexpr int kScale = 2 * kStep * kRow;
  static constexpr int kBytes = kScale + (kQ8 ? 2 * kStep * 4 : 0);
  static constexpr int kRing = kQ8 ? 4 : 2;          // steps of a warp's ring
  static constexpr int kBlock = kRowWarps * kRing * kBytes;
  static __device__ __forceinline__ int k_at(int key, int chunk) {
    return key * kRow + (kQ8 ? chunk : chunk ^ (key & 7)) * 16;
  }
  static __device__ __forceinline__ int v_at(int key, int chunk) {
    return kV + key * kRow + (kQ8 ? chunk ^ ((key >> 1) & 3) : chunk ^ (key & 7)) * 16;
  }
};

__device__ __forceinline__ void cp_async_or_zero16(uint32_t saddr, const void* g, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(g), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_or_zero4(uint32_t saddr, const void* g, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(saddr), "l"(g), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// (ordinary loads: the read-only path is for what no kernel writes while this one runs, and the one before may)
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  }
}

// Takes the non-finite values out of a pair (zero in their place); true if there was one.
template <typename T>
__device__ __forceinline__ bool take_nonfinite(uint32_t& x) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  const uint32_t bad = __vcmpeq2(x & kExp, kExp);
  x &= ~bad;
  return bad != 0;
}

// W warps share a unit of work (some rows, some keys): 1 where sequences are many and short, so that no warp waits
// for another, else the block's 4, whose parts are joined in shared memory first. MIXED: there are keys that some rows
// of a tile see and others do not, and their values may be infinite or NaN (beside the test for it in every kernel, 64
// sequences of one query took 31.3 us in place of 30.0).
template <typename T, int KIND, int MT, int W, bool MIXED>
__global__ void __launch_bounds__(kRowThreads, MT == 1 ? 3 : 2)
    attn_rows_kernel(PrefixArgs a, int prefix_tiles, int suffix_tiles, int prefix_units, int units, uint32_t* status,
                     bool after_tc) {
  extern __shared__ __align__(16) uint8_t s_ring[];
  using Mem = StepMem<KIND>;
  __shared__ int s_pages[W == 1 ? 1 : kMaxChunkPages];
  __shared__ __align__(16) float s_o[W == 1 ? 1 : W][W == 1 ? 1 : MT * 16][kPitch];
  __shared__ float2 s_ml[W][MT * 16];
  // After the tcgen05 kernel of the same call the inputs are complete already and no part is shared with it: this kernel
  // then waits for it only at the end, so that the join, which waits for this one, has both.
  if (after_tc)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  else
    pdl_enter();
  const int warp = W == 1 ? 0 : threadIdx.x >> 5;  // in the team
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y;
  int u = W == 1 ? blockIdx.x * kRowWarps + (threadIdx.x >> 5) : blockIdx.x;
  if (W == 1 && u >= units) {
    if (after_tc) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  // this unit's rows [row0, row_end), keys [first, end), page list and part
  const int span = a.q_len * a.group;
  int row0, row_end, first, end, part, b = 0;
  int len = 0;             // of the suffix of the rows' sequence
  int base_len = 1 << 30;  // keys that its last query sees
  const int32_t* list;
  const bool shared = u < prefix_units;
  if (shared) {
    part = prefix_tiles == 1 ? u : u / prefix_tiles;
    row0 = (u - part * prefix_tiles) * MT * 16;
    row_end = min(a.rows, row0 + MT * 16);
    first = part * a.prefix_chunk;
    end = min(a.prefix_len, first + a.prefix_chunk);
    list = a.prefix_pages;
  } else {
    u -= prefix_units;
    b = u / (a.n_suffix * suffix_tiles);
    u -= b * a.n_suffix * suffix_tiles;
    const int s = suffix_tiles == 1 ? u : u / suffix_tiles, tile = u - s * suffix_tiles;
    part = a.suffix_part + s;
    row0 = b * span + tile * MT * 16;
    row_end = min((b + 1) * span, row0 + MT * 16);
    first = s * a.suffix_chunk;
    end = min(a.max_suffix, first + a.suffix_chunk);  // (until the length is here)
    list = a.suffix_pages + (long long)b * a.suffix_pitch;
    len = suffix_len(a, b, status);
  }
  // the page list, the length and Q come together
  const int sh = a.c.page_shift;
  const int pages = ((end - 1) >> sh) - (first >> sh) + 1;
  int my_page = 0;  // (W 1: kSinglePages at most)
  if (W == 1) {
    if (lane < pages) my_page = list[(first >> sh) + lane];
  } else {
    for (int i = threadIdx.x; i < pages; i += kRowThreads) s_pages[i] = list[(first >> sh) + i];
  }
  // a page that the list has wrong: recorded, page 0 in its place
  auto checked = [&](int page, bool used) {
    const bool bad = (unsigned)page >= (unsigned)a.c.n_pages;
    if (bad && used) atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
    return bad ? 0 : page;
  };

  // Q fragments and the number of keys that each of the thread's rows sees (rows that do not exist see all)
  uint32_t q[MT][4][4];  // A fragments, [k step]
  int lim[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row0 + m * 16 + e * 8 + g;
      lim[m][e] = 1 << 30;
      uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (r < row_end) {
        const int token = r / a.group;
        const T* src = static_cast<const T*>(a.q) + (long long)token * a.ld_q +
                       (kvh * a.group + r - token * a.group) * kKvHeadDim + t * 16;
        load_words(w, reinterpret_cast<const uint8_t*>(src));
        if (!shared) lim[m][e] = (b + 1) * a.q_len - 1 - token;  // later queries: taken off the length below
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        q[m][k][e] = w[2 * k];
        q[m][k][2 + e] = w[2 * k + 1];
      }
    }
  if (!shared) {
    base_len = len;
    end = min(end, len);
    if (first >= end) {  // no key here
      if (after_tc) asm volatile("griddepcontrol.wait;" ::: "memory");
      return;
    }
  }
  int min_lim = 1 << 30;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (shared)
        lim[m][e] = end;
      else if (lim[m][e] < (1 << 30))
        lim[m][e] = min(end, base_len - lim[m][e]);
      else
        lim[m][e] = end;
      min_lim = min(min_lim, lim[m][e]);
    }
  // From here on some of the suffix's keys are seen by its later queries alone.
  const int first_hidden = shared ? 1 << 30 : len - (a.q_len - 1);
  const int used_pages = ((end - 1) >> sh) - (first >> sh) + 1;
  if (W == 1) {
    my_page = checked(my_page, lane < used_pages);
  } else {  // (each thread checks what it loaded)
    for (int i = threadIdx.x; i < used_pages; i += kRowThreads) s_pages[i] = checked(s_pages[i], true);
    __syncthreads();
  }

  float o[MT][8][4];
  float mx[MT][2], l[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mx[m][0] = mx[m][1] = -INFINITY;
    l[m][0] = l[m][1] = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
  }

  const uint32_t ring = smem_u32(s_ring) + (threadIdx.x >> 5) * (Mem::kRing * Mem::kBytes);
  const uint32_t page_vecs = (uint32_t)a.c.kv_heads << sh;  // vectors of a page (its bytes may pass 32 bits)
  const uint8_t* k0 = a.c.k + ((long long)kvh << sh) * Mem::kRow + lane * 16;
  const uint8_t* v0 = a.c.v + ((long long)kvh << sh) * Mem::kRow + lane * 16;
  auto page_of = [&](int key) {
    const int at = (min(key, end - 1) >> sh) - (first >> sh);
    return (uint32_t)(W == 1 ? __shfl_sync(~0u, my_page, at) : s_pages[at]);
  };
  // Step i of this warp: keys from first + (warp + i·W)·32 on, zeros past the end.
  auto fetch = [&](int i) {
    const int key0 = first + (warp + i * W) * kStep;
    if (key0 < end) {
      const uint32_t dst = ring + (i % Mem::kRing) * Mem::kBytes;
      const bool whole = key0 + kStep <= end;
      constexpr int kKeys = 32 / Mem::kChunks;  // keys of one round of the warp: 8 (8-bit kinds) or 4
#pragma unroll
      for (int n = 0; n < kStep / kKeys; ++n) {
        const int at = (key0 + n * kKeys) & ((1 << sh) - 1);  // (a round lies inside one page)
        const unsigned long long off = ((unsigned long long)page_of(key0 + n * kKeys) * page_vecs + at) * Mem::kRow;
        const int kk = n * kKeys + lane / Mem::kChunks, ch = lane % Mem::kChunks;
        const bool live = whole || key0 + kk < end;
        cp_async_or_zero16(dst + Mem::k_at(kk, ch), k0 + off, live);
        cp_async_or_zero16(dst + Mem::v_at(kk, ch), v0 + off, live);
      }
      if constexpr (Mem::kQ8) {
        const unsigned long long at = (unsigned long long)page_of(key0 + lane) * page_vecs + ((uint32_t)kvh << sh) +
                                      ((key0 + lane) & ((1 << sh) - 1));
        const bool live = whole || key0 + lane < end;
        cp_async_or_zero4(dst + Mem::kScale + lane * 4, a.c.k_scale + at, live);
        cp_async_or_zero4(dst + Mem::kScale + (kStep + lane) * 4, a.c.v_scale + at, live);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < Mem::kRing; ++i) fetch(i);
  for (int i = 0;; ++i) {
    const int key0 = first + (warp + i * W) * kStep;
    if (key0 >= end) break;
    cp_async_wait<Mem::kRing - 1>();
    __syncwarp();
    const uint32_t src = ring + (i % Mem::kRing) * Mem::kBytes;
    // S = Q·Kᵀ
    float s[MT][4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t kb[8];
      if constexpr (KIND == B2P_KV_16) {
        const uint4 x = lds16(src + Mem::k_at(8 * j + g, 2 * t)), y = lds16(src + Mem::k_at(8 * j + g, 2 * t + 1));
        kb[0] = x.x, kb[1] = x.y, kb[2] = x.z, kb[3] = x.w, kb[4] = y.x, kb[5] = y.y, kb[6] = y.z, kb[7] = y.w;
      } else {
        const uint4 x = lds16(src + Mem::k_at(8 * j + g, t));
        widen4<T, KIND>(x.x, kb[0], kb[1]);
        widen4<T, KIND>(x.y, kb[2], kb[3]);
        widen4<T, KIND>(x.z, kb[4], kb[5]);
        widen4<T, KIND>(x.w, kb[6], kb[7]);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        s[m][j][0] = s[m][j][1] = s[m][j][2] = s[m][j][3] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) mma16816<T>(s[m][j], q[m][k], kb[2 * k], kb[2 * k + 1]);
      }
    }
    // scores in the log2 domain, masked where a row's keys end; the value's scale joins in
    const bool whole = key0 + kStep <= min_lim;
    const bool mixed = MIXED && key0 + kStep > first_hidden;  // (the same in all lanes)
    float vi[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float kc[2] = {kScaleLog2, kScaleLog2}, vl[2] = {0.f, 0.f};
      if constexpr (KIND != B2P_KV_16) {
        const uint2 ks = lds8(src + Mem::kScale + (8 * j + 2 * t) * 4);
        const uint2 vs = lds8(src + Mem::kScale + (kStep + 8 * j + 2 * t) * 4);
        // A smaller scale, such as that of a vector of zeros, counts as 2^-80: then neither its logarithm nor its
        // reciprocal leaves fp32, and beside a scale of 2^30 (2^9 is fp16's most) only weights below 2^-16 of the largest
        // are lost from l. (A key that is not there has scale 0.)
        const float y0 = __uint_as_float(vs.x), y1 = __uint_as_float(vs.y);
        const float v0 = fabsf(y0) < 0x1p-80f ? 0x1p-80f : y0, v1 = fabsf(y1) < 0x1p-80f ? 0x1p-80f : y1;
        kc[0] = __uint_as_float(ks.x) * kScaleLog2;
        kc[1] = __uint_as_float(ks.y) * kScaleLog2;
        vl[0] = log2_sfu(v0);
        vl[1] = log2_sfu(v1);
        // (a NaN scale has the weights NaN already; where a row does not see the key, its weight of 0 must stay one)
        vi[j][0] = fmaxf(rcp_sfu(v0), 0.f);
        vi[j][1] = fmaxf(rcp_sfu(v1), 0.f);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[m][j][i] = KIND == B2P_KV_16 ? s[m][j][i] * kScaleLog2 : fmaf(s[m][j][i], kc[i & 1], vl[i & 1]);
        if (!whole) {
          const int key = key0 + 8 * j + 2 * t;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (key >= lim[m][e]) s[m][j][2 * e] = -INFINITY;
            if (key + 1 >= lim[m][e]) s[m][j][2 * e + 1] = -INFINITY;
          }
        }
      }
    }
    // the rows' references move, to the next integer above, only for a score more than kSlack above them
    bool up = false;
    float top[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(s[m][0][2 * e], s[m][0][2 * e + 1]);
#pragma unroll
        for (int j = 1; j < 4; ++j) x = fmaxf(x, fmaxf(s[m][j][2 * e], s[m][j][2 * e + 1]));
        top[m][e] = x;
        up = up || x > mx[m][e] + kSlack;
      }
    if (__any_sync(~0u, up)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = top[m][e];
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
          x = fmaxf(x, __shfl_xor_sync(~0u, x, 2));
          const float now = x > mx[m][e] + kSlack ? ceilf(x) : mx[m][e];
          const float f = now == mx[m][e] ? 1.f : exp2_sfu(mx[m][e] - now);
          mx[m][e] = now;
          l[m][e] *= f;
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            o[m][n][2 * e] *= f;
            o[m][n][2 * e + 1] *= f;
          }
        }
    }
    uint32_t pa[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ref = mx[m][e] == -INFINITY ? 0.f : mx[m][e];  // a row that sees none of the keys so far
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = exp2_sfu(s[m][j][2 * e] - ref), p1 = exp2_sfu(s[m][j][2 * e + 1] - ref);
          sum += KIND == B2P_KV_16 ? p0 + p1 : fmaf(p0, vi[j][0], p1 * vi[j][1]);
          pa[m][j >> 1][(j & 1) * 2 + e] = pack_h2<T>(p0, p1);
        }
        l[m][e] += sum;
      }
    // O += w·V: pairs (key 2t, key 2t + 1) of a tile, channel 8g + n
    bool odd = false;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      uint32_t vb[2][8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = 8 * (2 * jj + j) + 2 * t;
        if constexpr (KIND == B2P_KV_16) {
          const uint4 x = lds16(src + Mem::v_at(key, g)), y = lds16(src + Mem::v_at(key + 1, g));
          const uint32_t v[2][4] = {{x.x, x.y, x.z, x.w}, {y.x, y.y, y.z, y.w}};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vb[j][2 * i] = __byte_perm(v[0][i], v[1][i], 0x5410);
            vb[j][2 * i + 1] = __byte_perm(v[0][i], v[1][i], 0x7632);
          }
        } else {
          const uint2 x = lds8(src + Mem::v_at(key, g >> 1) + (g & 1) * 8);
          const uint2 y = lds8(src + Mem::v_at(key + 1, g >> 1) + (g & 1) * 8);
          widen4<T, KIND>(__byte_perm(x.x, y.x, 0x5140), vb[j][0], vb[j][1]);
          widen4<T, KIND>(__byte_perm(x.x, y.x, 0x7362), vb[j][2], vb[j][3]);
          widen4<T, KIND>(__byte_perm(x.y, y.y, 0x5140), vb[j][4], vb[j][5]);
          widen4<T, KIND>(__byte_perm(x.y, y.y, 0x7362), vb[j][6], vb[j][7]);
        }
      }
      if (mixed) {
#pragma unroll
        for (int n = 0; n < 8; ++n) odd |= take_nonfinite<T>(vb[0][n]) | take_nonfinite<T>(vb[1][n]);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 8; ++n) mma16816<T>(o[m][n], pa[m][jj], vb[0][n], vb[1][n]);
    }
    if (mixed && __any_sync(~0u, odd)) {
      // A product with a weight of 0 would bring a value that is not finite to rows that do not see it. Those values
      // were left out above; here the rows that see them get them. (A thread's columns of O: channels 16t + n and
      // 16t + 8 + n.)
#pragma unroll 1
      for (int k = 0; k < kStep; ++k) {
        uint32_t x[8];  // the channels' pairs
        if constexpr (KIND == B2P_KV_16) {
          const uint4 a0 = lds16(src + Mem::v_at(k, 2 * t)), a1 = lds16(src + Mem::v_at(k, 2 * t + 1));
          x[0] = a0.x, x[1] = a0.y, x[2] = a0.z, x[3] = a0.w, x[4] = a1.x, x[5] = a1.y, x[6] = a1.z, x[7] = a1.w;
        } else {
          const uint4 c = lds16(src + Mem::v_at(k, t));
          widen4<T, KIND>(c.x, x[0], x[1]);
          widen4<T, KIND>(c.y, x[2], x[3]);
          widen4<T, KIND>(c.z, x[4], x[5]);
          widen4<T, KIND>(c.w, x[6], x[7]);
        }
#pragma unroll
        for (int n = 0; n < 8; n += 2)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t rest = x[4 * c + n / 2];
            const float2 v = H2<T>::to_f2(*reinterpret_cast<typename H2<T>::V*>(&x[4 * c + n / 2]));
            if (!take_nonfinite<T>(rest)) continue;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (key0 + k >= lim[m][e]) continue;
                if (!(fabsf(v.x) < INFINITY)) o[m][n][2 * e + c] += v.x;
                if (!(fabsf(v.y) < INFINITY)) o[m][n + 1][2 * e + c] += v.y;
              }
          }
      }
    }
    __syncwarp();
    fetch(i + Mem::kRing);
  }

  const int count = row_end - row0;
  const long long at0 = ((long long)part * a.c.kv_heads + kvh) * a.rows + row0;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[m][e];
      sum += __shfl_xor_sync(~0u, sum, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      const int r = m * 16 + e * 8 + g;
      if (r < count) {
        if (t == 0) (W == 1 ? a.part_ml[at0 + r] : s_ml[warp][r]) = make_float2(mx[m][e], sum);
        float* dst = (W == 1 ? a.part_o + (at0 + r) * kKvHeadDim : &s_o[warp][r][0]) + 16 * t;
#pragma unroll
        for (int n = 0; n < 8; n += 4) {
          *reinterpret_cast<float4*>(dst + n) =
              make_float4(o[m][n][2 * e], o[m][n + 1][2 * e], o[m][n + 2][2 * e], o[m][n + 3][2 * e]);
          *reinterpret_cast<float4*>(dst + 8 + n) =
              make_float4(o[m][n][2 * e + 1], o[m][n + 1][2 * e + 1], o[m][n + 2][2 * e + 1], o[m][n + 3][2 * e + 1]);
        }
      }
    }
  if (W > 1) {  // join the warps' parts
    __syncthreads();
    for (int i = threadIdx.x; i < count * 16; i += kRowThreads) {
      const int r = i >> 4, d = (i & 15) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][r].x);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = exp2_sfu(s_ml[w][r].x - ref);
        sum += f * s_ml[w][r].y;
        const float4 x = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
      }
      *reinterpret_cast<float4*>(a.part_o + (at0 + r) * kKvHeadDim + d) = acc;
      if (d == 0) a.part_ml[at0 + r] = make_float2(top, sum);
    }
  }
  if (after_tc) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A half warp per row: join the row's parts (zeros where there is none).
template <typename T>
__global__ void __launch_bounds__(128) attn_join_kernel(PrefixArgs a, uint32_t* status) {
  pdl_enter();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 4);
  if (r >= a.rows) return;
  const int len = a.suffix_lens ? suffix_len(a, r / (a.q_len * a.group), status) : 0;
  join_row<T>(a, blockIdx.y, r, len, threadIdx.x & 15);
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// How the work is divided: about four blocks for each SM, no part shorter than kMinPart keys nor
// longer than the page list that a block keeps.
struct Plan {
  bool tc;  // the prefix goes to the tcgen05 kernel
  int team;  // warps that share a unit of attn_rows_kernel
  int mt, prefix_tiles, suffix_tiles, n_suffix, suffix_chunk;
  PrefixSplit split;
  int suffix_part, parts;
};
int chunk_for(int len, int tiles, int want) {
  int n = ceil_div(want, tiles);
  const int most = ceil_div(len, kMinPart);
  if (n > most) n = most;
  if (n < 1) n = 1;
  int chunk = ceil_div(ceil_div(len, n), kMinPart) * kMinPart;
  return chunk > kMaxChunk ? kMaxChunk : chunk;
}
int single_chunk(int len) {  // keys of a single warp's unit: about eight units, of 128 to 1024 keys
  int chunk = kMinPart;
  while (chunk < 1024 && chunk * 8 < len) chunk *= 2;
  return chunk;
}
Plan make_plan(int batch, int q_len, int group, int prefix_len, int max_suffix, const KvView& c) {
  Plan p = {};
  const int rows = batch * q_len * group, kv_heads = c.kv_heads;
  p.tc = prefix_len >= kTcKeys || (long long)rows * prefix_len >= (c.kind == B2P_KV_16 ? kTcWork16 : kTcWork8);
  p.mt = (p.tc || prefix_len == 0 ? q_len * group : rows) > 16 ? 2 : 1;
  p.prefix_tiles = ceil_div(rows, 16 * p.mt);
  p.suffix_tiles = ceil_div(q_len * group, 16 * p.mt);
  p.team = kRowWarps;
  p.split.pair_rows = rows;
  if (p.tc) {
    prefix_tc_plan(rows, kv_heads, prefix_len, &p.split);
  } else if (prefix_len > 0) {
    p.split.prefix_chunk = chunk_for(prefix_len, p.prefix_tiles * kv_heads, kWant);
    p.split.n_prefix = ceil_div(prefix_len, p.split.prefix_chunk);
  }
  if (max_suffix > 0) {
    const long long teams = (long long)batch * p.suffix_tiles * kv_heads;
    p.suffix_chunk = chunk_for(max_suffix, (int)(teams < kWant ? teams : kWant), kWant);
    // Units of single warps where there are sequences enough to fill the GPU with them. Measured, 5 KV heads, teams of 4 /
    // single warps: suffixes of 1000 alone, 8 sequences 9.6 / 9.1 us, 16 12.6 / 10.7, 64 22.7 / 16.1; of 8000, 16
    // sequences 33 / 47, 32 55 / 51, 64 94 / 81; 32 sequences of 500 after 500 shared keys 14.5 / 12.8, 16 of 300 after
    // 1000 10.7 / 11.4. Units of 128, 256, 512 keys for 256 suffixes of 512: 40 / 39 / 43, for 128 of 4096 101 / 88 / 84.
    const int chunk = single_chunk(max_suffix), shared_chunk = single_chunk(p.tc ? 0 : prefix_len);
    const bool many = teams >= kSms || ((p.tc || prefix_len == 0) && 2 * teams >= kSms && max_suffix <= 2048);
    if (many && max(chunk, shared_chunk) <= kSinglePages << c.page_shift) {
      p.team = 1;
      p.suffix_chunk = chunk;
      if (!p.tc && prefix_len > 0) {
        p.split.prefix_chunk = shared_chunk;
        p.split.n_prefix = ceil_div(prefix_len, shared_chunk);
      }
    }
    p.n_suffix = ceil_div(max_suffix, p.suffix_chunk);
  }
  p.suffix_part = p.split.n_prefix > p.split.n_last ? p.split.n_prefix : p.split.n_last;
  p.parts = p.suffix_part + p.n_suffix;
  return p;
}

template <typename T, int KIND, int MT, int W, bool MIXED>
int launch_rows(const PrefixArgs& a, const Plan& p, const DeviceCtx* c, cudaStream_t st) {
  const long long prefix_units = p.tc ? 0 : (long long)p.split.n_prefix * p.prefix_tiles;
  const long long units = prefix_units + (long long)a.batch * p.n_suffix * p.suffix_tiles;
  B2P_REQUIRE(units < (1ll << 31), "too much work for one call");
  static thread_local uint64_t attr_mask = 0;  // one per instantiation
  constexpr int kSmem = StepMem<KIND>::kBlock;
  const auto kernel = attn_rows_kernel<T, KIND, MT, W, MIXED>;
  if (!(attr_mask & (1ull << (c->device & 63)))) {
    B2P_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    attr_mask |= 1ull << (c->device & 63);
  }
  const int blocks = W == 1 ? ceil_div((int)units, kRowWarps) : (int)units;
  B2P_CHECK_CUDA(launch_pdl(kernel, dim3(blocks, a.c.kv_heads), dim3(kRowThreads), kSmem, st, a, p.prefix_tiles,
                            p.suffix_tiles, (int)prefix_units, (int)units, c->status, p.tc));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

template <typename T, int KIND, bool MIXED>
int launch_w(const PrefixArgs& a, const Plan& p, const DeviceCtx* c, cudaStream_t st) {
  if (p.team == 1)
    return p.mt == 2 ? launch_rows<T, KIND, 2, 1, MIXED>(a, p, c, st) : launch_rows<T, KIND, 1, 1, MIXED>(a, p, c, st);
  return p.mt == 2 ? launch_rows<T, KIND, 2, kRowWarps, MIXED>(a, p, c, st)
                   : launch_rows<T, KIND, 1, kRowWarps, MIXED>(a, p, c, st);
}

template <typename T, int KIND>
int run_t(const PrefixArgs& a, const Plan& p, const DeviceCtx* c, cudaStream_t st) {
  int rc = B2P_OK;
  if (p.tc) rc = launch_prefix_tc(a, std::is_same<T, __nv_bfloat16>::value, st);
  if (rc) return rc;
  if (p.n_suffix > 0 || (p.split.n_prefix > 0 && !p.tc)) {
    constexpr bool kFinite = KIND == B2P_KV_INT8;  // whatever the codes
    rc = kFinite || p.n_suffix == 0 || a.q_len == 1 ? launch_w<T, KIND, false>(a, p, c, st)
                                                    : launch_w<T, KIND, !kFinite>(a, p, c, st);
  }
  if (rc) return rc;
  B2P_CHECK_CUDA(launch_pdl(attn_join_kernel<T>, dim3(ceil_div(a.rows, 8), a.c.kv_heads), dim3(128), 0, st, a,
                            c->status));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

template <typename T>
int run_kind(const PrefixArgs& a, const Plan& p, const DeviceCtx* c, cudaStream_t st) {
  switch (a.c.kind) {
    case B2P_KV_INT8:
      return run_t<T, B2P_KV_INT8>(a, p, c, st);
    case B2P_KV_E4M3:
      return run_t<T, B2P_KV_E4M3>(a, p, c, st);
    default:
      return run_t<T, B2P_KV_16>(a, p, c, st);
  }
}

bool sizes_ok(int batch, int q_len, int heads, int kv_heads, int prefix_len, int max_suffix) {
  return batch >= 1 && q_len >= 1 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && kv_heads <= 65535 &&
         prefix_len >= 0 && max_suffix >= 0 && prefix_len <= (1 << 30) && max_suffix <= (1 << 30) &&
         (long long)batch * q_len * heads < (1ll << 30);
}

}  // namespace
}  // namespace b2p

using namespace b2p;

extern "C" {

size_t b2p_attention_prefix_workspace(int batch, int q_len, int heads, int kv_heads, int prefix_len, int max_suffix) {
  if (!sizes_ok(batch, q_len, heads, kv_heads, prefix_len, max_suffix)) return 0;
  // A bound that grows with every argument, so that the workspace of the largest call serves all: parts are
  // kTcStageKeys keys or longer, and there are about kWant blocks of 32 rows, or kSms of 256, or one per kMaxChunk keys,
  // or single-warp units: at most 8 a row, or of 1024 keys.
  const long long rows = (long long)batch * q_len * heads;
  long long slots = 0;
  for (int len : {prefix_len, max_suffix}) {
    if (len == 0) continue;
    const long long by_length = rows * ceil_div(len, kTcStageKeys);
    const long long by_blocks = (long long)kSms * 256 + rows * (10 + len / 1024);
    slots += by_length < by_blocks ? by_length : by_blocks;
  }
  return (size_t)slots * (kKvHeadDim * sizeof(float) + sizeof(float2)) + 256;
}

int b2p_attention_prefix(const b2p_kv_cache* cache, const void* q, int ld_q, void* out, int ld_out, float* lse,
                         int batch, int q_len, int heads, const int32_t* prefix_pages, int prefix_len,
                         const int32_t* suffix_pages, int suffix_pitch, const int32_t* suffix_lens, int max_suffix,
                         int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  PrefixArgs a;
  int rc = kv_view(cache, dtype, &a.c);
  if (rc) return rc;
  B2P_REQUIRE(heads >= 1 && heads % a.c.kv_heads == 0, "heads (%d) must be a multiple of kv_heads (%d)", heads,
              a.c.kv_heads);
  B2P_REQUIRE(sizes_ok(batch, q_len, heads, a.c.kv_heads, prefix_len, max_suffix),
              "batch, q_len, prefix_len or max_suffix out of range");
  B2P_REQUIRE(q && out, "null q or out");
  for (int ld : {ld_q, ld_out})
    B2P_REQUIRE(ld >= heads * kKvHeadDim && ld % 8 == 0, "q and out rows must hold %d columns and keep 16-byte rows",
                heads * kKvHeadDim);
  B2P_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0,
              "q and out must be 16-byte aligned");
  B2P_REQUIRE(prefix_len == 0 || prefix_pages, "null prefix_pages");
  if (max_suffix > 0) {
    B2P_REQUIRE(suffix_pages && suffix_lens, "null suffix_pages or suffix_lens");
    B2P_REQUIRE(suffix_pitch >= ceil_div(max_suffix, cache->page_size), "suffix_pitch (%d) does not hold %d tokens",
                suffix_pitch, max_suffix);
  }
  const size_t need = b2p_attention_prefix_workspace(batch, q_len, heads, a.c.kv_heads, prefix_len, max_suffix);
  B2P_REQUIRE(workspace && workspace_bytes >= need, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  B2P_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "workspace must be 16-byte aligned");
  const int group = heads / a.c.kv_heads;
  const Plan p = make_plan(batch, q_len, group, prefix_len, max_suffix, a.c);
  const size_t all_rows = (size_t)batch * q_len * heads;
  const size_t uses = (size_t)p.parts * all_rows * (kKvHeadDim * sizeof(float) + sizeof(float2));
  B2P_REQUIRE(uses <= workspace_bytes, "workspace bound of %zu bytes does not hold %zu", need, uses);
  DeviceCtx* c = nullptr;
  if ((rc = ctx_get(&c))) return rc;
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.prefix_pages = prefix_pages;
  a.suffix_pages = suffix_pages;
  a.suffix_lens = suffix_lens;
  a.rows = batch * q_len * group;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o +
                                        (size_t)p.parts * a.rows * a.c.kv_heads * kKvHeadDim);
  a.ld_q = ld_q;
  a.ld_out = ld_out;
  a.batch = batch;
  a.q_len = q_len;
  a.group = group;
  a.prefix_len = prefix_len;
  a.suffix_pitch = suffix_pitch;
  a.max_suffix = max_suffix;
  static_cast<PrefixSplit&>(a) = p.split;
  a.suffix_part = p.suffix_part;
  a.n_suffix = p.n_suffix;
  a.suffix_chunk = p.suffix_chunk > 0 ? p.suffix_chunk : 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == B2P_BF16 ? run_kind<__nv_bfloat16>(a, p, c, st) : run_kind<__half>(a, p, c, st);
}

}  // extern "C"
