// attn_prefix.cu — attention of a batch that shares a long prefix, over a paged
// cache of 16-bit or 8-bit keys and values.
//
// With s_j = q·k_j / 8 and any split of a row's keys into parts, each part's
//   m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j
// join to out = sum e^(m_p - M) o_p / sum e^(m_p - M) l_p, M = max m_p, and the
// log-sum-exp M + log(sum e^(m_p - M) l_p). The shared prefix is one part list
// for the rows of all sequences at once (its keys are read once for the batch);
// each sequence's suffix is another.
//
// attn_rows_kernel: each warp holds 16 or 32 query rows of one KV head and runs
// over 32 keys at a time with mma.sync. Keys and values go from global memory
// straight into the registers of the fragment: a head's 64 channels are taken in
// the order that gives each thread 16 consecutive ones of a key (S = Q·Kᵀ sums
// over channels, so Q is read in the same order) and 8 consecutive ones of a
// value (each is a column of O of its own).
//
// 8-bit caches: codes widen to 16 bit exactly. A key's scale multiplies its
// column of S in fp32. A value's scale y_j joins the exponent,
//   w_j = exp2(s_j log2e + log2 y_j - M), M the running maximum of the sum,
// so that o = sum w_j code_j, l = sum w_j / y_j and out = o / l: the one rounding
// to 16 bit is that of w_j <= 1, as without scales, however small the values are.
#include <cstdint>
#include <type_traits>
#include "attn_prefix.cuh"
#include "ptx.cuh"

namespace b2p {
namespace {

constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kStep = 32;            // keys of one warp step
constexpr int kMaxChunk = 4096;      // keys of one part
constexpr int kMaxChunkPages = kMaxChunk / 8 + 1;
constexpr int kMinPart = 128;        // no part shorter: its join would cost what it saves
constexpr int kWant = kSms * 4;      // blocks wanted of each list
constexpr int kTcRows = 64;          // rows from which the prefix goes to the tcgen05 kernel

__device__ __forceinline__ float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_sfu(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Keys of one step as loaded: n8 tiles j = 0..3 of 8 keys each.
template <int KIND>
struct StepRegs {
  static constexpr int kKW = KIND == B2P_KV_16 ? 8 : 4;  // words of a thread's 16 channels of a key
  static constexpr int kVW = KIND == B2P_KV_16 ? 4 : 2;  // words of its 8 channels of a value
  uint32_t k[4][kKW];
  uint32_t v[4][2][kVW];
  float2 ks[4], vs[4];
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 2) {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = x.x;
    w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  }
}

// Load the 32 keys from key0 (a multiple of 8 inside the list) on; keys from `end` on give zeros.
// pages[] is the part's page list in shared memory, its first page holding key `first`.
template <int KIND>
__device__ __forceinline__ void load_step(StepRegs<KIND>& r, const KvView& c, const int* pages, int first, int kvh,
                                          int key0, int end, int g, int t) {
  constexpr int kBytes = KIND == B2P_KV_16 ? 128 : 64;  // of a key
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int key = key0 + 8 * j;
#pragma unroll
    for (int i = 0; i < StepRegs<KIND>::kKW; ++i) r.k[j][i] = 0;
#pragma unroll
    for (int i = 0; i < StepRegs<KIND>::kVW; ++i) r.v[j][0][i] = r.v[j][1][i] = 0;
    r.ks[j] = make_float2(0.f, 0.f);
    r.vs[j] = make_float2(1.f, 1.f);
    if (key >= end) continue;
    const int page = pages[(key >> c.page_shift) - (first >> c.page_shift)];
    if (page < 0) continue;
    const long long at = c.vec(page, kvh, key & ((1 << c.page_shift) - 1));
    if (key + g < end) load_words(r.k[j], c.k + (at + g) * kBytes + t * (kBytes / 4));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int kk = 2 * t + e;
      if (key + kk < end) {
        load_words(r.v[j][e], c.v + (at + kk) * kBytes + g * (kBytes / 8));
        if (KIND != B2P_KV_16) {
          (e ? r.ks[j].y : r.ks[j].x) = __ldg(c.k_scale + at + kk);
          (e ? r.vs[j].y : r.vs[j].x) = __ldg(c.v_scale + at + kk);
        }
      }
    }
  }
}

template <typename T, int KIND, int MT>
__global__ void __launch_bounds__(kRowThreads) attn_rows_kernel(PrefixArgs a, int prefix_tiles, int suffix_tiles,
                                                                int prefix_units, int overlap, uint32_t* status) {
  __shared__ int s_pages[kMaxChunkPages];
  __shared__ __align__(16) float s_o[kRowWarps][MT * 16][kKvHeadDim];
  __shared__ float2 s_ml[kRowWarps][MT * 16];
  // After the tcgen05 kernel of the same call (overlap) the inputs are complete already and no part is shared with
  // it: this kernel then waits for it only at the end, so that whoever waits for this one has both.
  if (overlap)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  else
    pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y;
  int u = blockIdx.x;
  // this block's rows [row0, row_end), keys [first, end), page list and part
  int row0, row_end, first, end, part;
  int base_len = 1 << 30;  // keys that the last query of the rows' sequence sees
  const int32_t* list;
  if (u < prefix_units) {
    part = u / prefix_tiles;
    row0 = (u % prefix_tiles) * MT * 16;
    row_end = min(a.rows, row0 + MT * 16);
    first = part * a.prefix_chunk;
    end = min(a.prefix_len, first + a.prefix_chunk);
    list = a.prefix_pages;
  } else {
    u -= prefix_units;
    const int per = a.n_suffix * suffix_tiles;
    const int b = u / per, s = (u % per) / suffix_tiles, tile = u % suffix_tiles;
    const int span = a.q_len * a.group;
    part = a.suffix_part + s;
    row0 = b * span + tile * MT * 16;
    row_end = min((b + 1) * span, row0 + MT * 16);
    first = s * a.suffix_chunk;
    base_len = suffix_len(a, b, status);
    end = min(base_len, first + a.suffix_chunk);
    list = a.suffix_pages + (long long)b * a.suffix_pitch;
    if (first >= end) {
      if (overlap) asm volatile("griddepcontrol.wait;" ::: "memory");
      return;
    }
  }
  const int sh = a.c.page_shift;
  for (int i = threadIdx.x; i <= ((end - 1) >> sh) - (first >> sh); i += kRowThreads) {
    int p = list[(first >> sh) + i];
    if (p < 0 || p >= a.c.n_pages) {
      atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
      p = -1;
    }
    s_pages[i] = p;
  }
  __syncthreads();

  // Q fragments and the number of keys that each of the thread's rows sees
  uint32_t q[MT][2][8];
  int lim[MT][2];
  int min_lim = 1 << 30;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row0 + m * 16 + e * 8 + g;
      lim[m][e] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) q[m][e][i] = 0;
      if (r < row_end) {
        const T* src = static_cast<const T*>(a.q) + (long long)(r / a.group) * a.ld_q +
                       (kvh * a.group + r % a.group) * kKvHeadDim + t * 16;
        load_words(q[m][e], reinterpret_cast<const uint8_t*>(src));
        lim[m][e] = min(end, base_len - (a.q_len - 1 - (r / a.group) % a.q_len));
      }
      min_lim = min(min_lim, lim[m][e]);
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

  StepRegs<KIND> cur;
  int key0 = first + warp * kStep;
  if (key0 < end) load_step<KIND>(cur, a.c, s_pages, first, kvh, key0, end, g, t);
  for (; key0 < end; key0 += kRowWarps * kStep) {
    // S = Q·Kᵀ
    float s[MT][4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t kb[8];
      if constexpr (KIND == B2P_KV_16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) kb[i] = cur.k[j][i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) widen4<T, KIND>(cur.k[j][i], kb[2 * i], kb[2 * i + 1]);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        s[m][j][0] = s[m][j][1] = s[m][j][2] = s[m][j][3] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t qa[4] = {q[m][0][2 * k], q[m][1][2 * k], q[m][0][2 * k + 1], q[m][1][2 * k + 1]};
          mma16816<T>(s[m][j], qa, kb[2 * k], kb[2 * k + 1]);
        }
      }
    }
    // V of the step as B fragments: pair (key 2t, key 2t + 1) of tile j, channel 8g + n
    uint32_t vb[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (KIND == B2P_KV_16) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[e][i] = cur.v[j][e][i];
        } else {
          widen4<T, KIND>(cur.v[j][e][0], w[e][0], w[e][1]);
          widen4<T, KIND>(cur.v[j][e][1], w[e][2], w[e][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vb[j][2 * i] = __byte_perm(w[0][i], w[1][i], 0x5410);
        vb[j][2 * i + 1] = __byte_perm(w[0][i], w[1][i], 0x7632);
      }
    }
    float kc[4][2], vl[4][2], vi[4][2];  // per key: factor of S, log2 of the value's scale, its inverse
    if constexpr (KIND != B2P_KV_16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        kc[j][0] = cur.ks[j].x * kScaleLog2;
        kc[j][1] = cur.ks[j].y * kScaleLog2;
        vl[j][0] = log2_sfu(cur.vs[j].x);
        vl[j][1] = log2_sfu(cur.vs[j].y);
        vi[j][0] = __frcp_rn(cur.vs[j].x);
        vi[j][1] = __frcp_rn(cur.vs[j].y);
      }
    }
    const int next = key0 + kRowWarps * kStep;
    if (next < end) load_step<KIND>(cur, a.c, s_pages, first, kvh, next, end, g, t);

    // scores in the log2 domain, masked where a row's keys end
    const bool whole = key0 + kStep <= min_lim;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[m][j][i] = KIND == B2P_KV_16 ? s[m][j][i] * kScaleLog2 : fmaf(s[m][j][i], kc[j][i & 1], vl[j][i & 1]);
        if (!whole) {
          const int key = key0 + 8 * j + 2 * t;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (key >= lim[m][e]) s[m][j][2 * e] = -INFINITY;
            if (key + 1 >= lim[m][e]) s[m][j][2 * e + 1] = -INFINITY;
          }
        }
      }
      uint32_t pa[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(s[m][j][2 * e], s[m][j][2 * e + 1]));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        const float now = fmaxf(mx[m][e], top);
        const float ref = now == -INFINITY ? 0.f : now;  // a row that sees none of the keys so far
        const float scale = exp2_sfu(mx[m][e] - ref);
        mx[m][e] = now;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = exp2_sfu(s[m][j][2 * e] - ref), p1 = exp2_sfu(s[m][j][2 * e + 1] - ref);
          sum += KIND == B2P_KV_16 ? p0 + p1 : fmaf(p0, vi[j][0], p1 * vi[j][1]);
          pa[j >> 1][(j & 1) * 2 + e] = pack_h2<T>(p0, p1);
        }
        l[m][e] = l[m][e] * scale + sum;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          o[m][n][2 * e] *= scale;
          o[m][n][2 * e + 1] *= scale;
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        mma16816<T>(o[m][n], pa[0], vb[0][n], vb[1][n]);
        mma16816<T>(o[m][n], pa[1], vb[2][n], vb[3][n]);
      }
    }
  }

  // join the warps' parts
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[m][e];
      sum += __shfl_xor_sync(~0u, sum, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      const int r = m * 16 + e * 8 + g;
      if (t == 0) s_ml[warp][r] = make_float2(mx[m][e], sum);
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        s_o[warp][r][16 * t + n] = o[m][n][2 * e];
        s_o[warp][r][16 * t + 8 + n] = o[m][n][2 * e + 1];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 16 * 16; i += kRowThreads) {
    const int r = i >> 4, d = (i & 15) * 4;
    if (row0 + r >= row_end) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, s_ml[w][r].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = exp2_sfu(s_ml[w][r].x - ref);
      sum += f * s_ml[w][r].y;
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      acc.x += f * x.x;
      acc.y += f * x.y;
      acc.z += f * x.z;
      acc.w += f * x.w;
    }
    const long long at = ((long long)part * gridDim.y + kvh) * a.rows + row0 + r;
    *reinterpret_cast<float4*>(a.part_o + at * kKvHeadDim + d) = acc;
    if (d == 0) a.part_ml[at] = make_float2(top, sum);
  }
  if (overlap) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One half-warp per row: join the row's parts, normalise, round.
template <typename T>
__global__ void __launch_bounds__(128) attn_join_kernel(PrefixArgs a, uint32_t* status) {
  pdl_enter();
  const int heads_kv = gridDim.y, kvh = blockIdx.y;
  const int r = blockIdx.x * 8 + (threadIdx.x >> 4), d = (threadIdx.x & 15) * 4;
  if (r >= a.rows) return;
  const int token = r / a.group;
  const int len = a.max_suffix > 0 ? suffix_len(a, token / a.q_len, status) : 0;
  const int used = a.max_suffix > 0 ? (len + a.suffix_chunk - 1) / a.suffix_chunk : 0;
  const int shared = r < a.pair_rows ? a.n_prefix : a.n_last;
  const int parts = shared + used;
  auto part = [&](int p) { return p < shared ? p : p - shared + a.suffix_part; };
  const long long stride = (long long)heads_kv * a.rows, at0 = (long long)kvh * a.rows + r;
  float top = -INFINITY;
  for (int p = 0; p < parts; ++p) top = fmaxf(top, a.part_ml[part(p) * stride + at0].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = 0; p < parts; ++p) {
    const float2 ml = a.part_ml[part(p) * stride + at0];
    const float f = exp2_sfu(ml.x - ref);
    sum += f * ml.y;
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + (part(p) * stride + at0) * kKvHeadDim + d);
    acc.x += f * x.x;
    acc.y += f * x.y;
    acc.z += f * x.z;
    acc.w += f * x.w;
  }
  const float inv = top == -INFINITY ? 0.f : 1.f / sum;
  const int h = kvh * a.group + r % a.group;
  T* out = static_cast<T*>(a.out) + (long long)token * a.ld_out + h * kKvHeadDim + d;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_h2<T>(acc.x * inv, acc.y * inv), pack_h2<T>(acc.z * inv, acc.w * inv));
  if (a.lse && d == 0) a.lse[(long long)token * heads_kv * a.group + h] = top == -INFINITY ? -INFINITY : ref + log2f(sum);
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// How the work is divided: about four blocks for each SM, no part shorter than kMinPart keys nor
// longer than the page list that a block keeps.
struct Plan {
  bool tc;  // the prefix goes to the tcgen05 kernel
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
Plan make_plan(int batch, int q_len, int group, int kv_heads, int prefix_len, int max_suffix) {
  Plan p = {};
  const int rows = batch * q_len * group;
  p.tc = prefix_len > 0 && rows >= kTcRows;
  p.mt = (p.tc || prefix_len == 0 ? q_len * group : rows) > 16 ? 2 : 1;
  p.prefix_tiles = ceil_div(rows, 16 * p.mt);
  p.suffix_tiles = ceil_div(q_len * group, 16 * p.mt);
  p.split.pair_rows = rows;
  if (p.tc) {
    prefix_tc_plan(rows, kv_heads, prefix_len, &p.split);
  } else if (prefix_len > 0) {
    p.split.prefix_chunk = chunk_for(prefix_len, p.prefix_tiles * kv_heads, kWant);
    p.split.n_prefix = ceil_div(prefix_len, p.split.prefix_chunk);
  }
  if (max_suffix > 0) {
    p.suffix_chunk = chunk_for(max_suffix, batch * p.suffix_tiles * kv_heads, kWant);
    p.n_suffix = ceil_div(max_suffix, p.suffix_chunk);
  }
  p.suffix_part = p.split.n_prefix > p.split.n_last ? p.split.n_prefix : p.split.n_last;
  p.parts = p.suffix_part + p.n_suffix;
  return p;
}

template <typename T, int KIND, int MT>
int launch_rows(const PrefixArgs& a, const Plan& p, const DeviceCtx* c, cudaStream_t st) {
  const long long prefix_units = p.tc ? 0 : (long long)p.split.n_prefix * p.prefix_tiles;
  const long long units = prefix_units + (long long)a.batch * p.n_suffix * p.suffix_tiles;
  B2P_REQUIRE(units < (1ll << 31), "too much work for one call");
  B2P_CHECK_CUDA(launch_pdl(attn_rows_kernel<T, KIND, MT>, dim3((unsigned)units, a.c.kv_heads), dim3(kRowThreads), 0,
                            st, a, p.prefix_tiles, p.suffix_tiles, (int)prefix_units, p.tc ? 1 : 0, c->status));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

template <typename T, int KIND>
int run_t(const PrefixArgs& a, const Plan& p, const DeviceCtx* c, cudaStream_t st) {
  int rc = B2P_OK;
  if (p.tc) rc = launch_prefix_tc(a, std::is_same<T, __nv_bfloat16>::value, st);
  if (rc) return rc;
  if (p.n_suffix > 0 || (p.split.n_prefix > 0 && !p.tc))
    rc = p.mt == 2 ? launch_rows<T, KIND, 2>(a, p, c, st) : launch_rows<T, KIND, 1>(a, p, c, st);
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
  // kTcStageKeys keys or longer, and there are about kWant blocks of 32 rows, or kSms of 256, or one per kMaxChunk keys.
  const long long rows = (long long)batch * q_len * heads;
  long long slots = 0;
  for (int len : {prefix_len, max_suffix}) {
    if (len == 0) continue;
    const long long by_length = rows * ceil_div(len, kTcStageKeys);
    const long long by_blocks = (long long)kSms * 256 + rows * (2 + len / kMaxChunk);
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
  const Plan p = make_plan(batch, q_len, group, a.c.kv_heads, prefix_len, max_suffix);
  const size_t uses = (size_t)p.parts * batch * q_len * heads * (kKvHeadDim * 4 + sizeof(float2));
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
  a.suffix_chunk = p.suffix_chunk;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == B2P_BF16 ? run_kind<__nv_bfloat16>(a, p, c, st) : run_kind<__half>(a, p, c, st);
}

}  // extern "C"
