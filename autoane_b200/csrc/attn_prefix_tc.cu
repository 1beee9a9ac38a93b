// attn_prefix_tc.cu — the prefix part of attention over a shared prefix on the
// tcgen05 tensor cores, in tiles of 128 rows (sequences x queries x query heads of
// one KV head). attn_prefix.cu has the formulas, the parts, the join and the rule
// by which a prefix comes here.
//
// A CTA takes one part of the prefix for two row tiles, or for the one left over
// when their number is odd. Keys and values come in stages of 128, widened to 16
// bit once for all its rows. Two streams of four softmax warps work on units of
// 128 rows x 64 keys: a row tile each, or every other unit of one row tile. A
// stream has 256 TMEM columns, three score buffers of 64 and O in 64; per unit:
//   S issuer:  S = Q·Kᵀ  (tcgen05.mma 128 x 64, K 64) into a buffer, two units ahead
//   softmax:   w_j = exp2(s_j - ref), one pass over S, the next 32 keys' scores being
//              read meanwhile; a warp has the 32 rows of its lane quarter and writes
//              16-bit w over columns [0, 32) of the buffer
//   O issuer:  O += w·V  (A from TMEM, V MN-major)
// The exponentials bound it (16 a cycle and SM; 64 channels give only 256 MACs of
// tensor work to each), and after them the issue of all the instructions around
// them. Row r of a tile is lane 32 (r % 4) + r / 4: the rows of a tile that is not
// full are spread over the SM's four sub-partitions, and with 64 rows or fewer the
// upper 16 lanes of each quarter are left out. Measured: 768 rows of 5 KV heads over
// 32768 int8 keys 70 us (28 us of exponentials; two warps share a scheduler's unit
// and weigh at 68% of its rate), 320 rows of 6 over 4001 16-bit keys 12.5 us, 64 rows
// of 12 over 8192 e4m3 keys 16 us.
//
// ref need not be the maximum: any number near it gives the same quotient. It is
// the next integer above the first unit's scores, and moves only when a unit's sum
// of weights passes 512 (until then each fits 16 bit easily); the sums are then
// scaled by a power of two and the unit is done again. So S is read once, no
// maximum is taken in the loop, and O stays in TMEM.
//
// 8-bit caches: a key's scale multiplies its column of S in fp32 (the log-sum-exp
// stays exact to fp32). A value's scale is 2^e·f, f in [1, 2): 2^e goes into the
// widened value, exactly but for e4m3 codes under fp16 that fall below 2^-24 (they are
// off by 2^-25 at most, as an fp16 output of their size would be), and f into w before
// its one rounding; the sum of the
// weights is taken without it. S is read as 16 lanes x 256 bit, which gives a
// thread four rows and a quarter of the columns: a column's factors are read from
// shared memory once for four scores.
//
// Warps 0-3 load: 8-bit codes by cp.async three stages ahead into a raw ring,
// then through registers into the 128-byte-swizzled operand tiles (each thread
// widens what it loaded); 16-bit ones by cp.async straight into the tiles.
#include <cstdint>
#include <type_traits>
#include "attn_prefix.cuh"
#include "ptx.cuh"

namespace b2p {
namespace {

constexpr int kTcThreads = 512;
constexpr int kSoftWarp0 = 4, kIssueWarp0 = 12;
constexpr int kTileRows = 128;
constexpr int kStageKeys = kTcStageKeys;
constexpr int kUnitKeys = 64;
constexpr int kBufs = 3;                                 // score buffers of a stream
constexpr int kOCol = kBufs * kUnitKeys;                 // O in a stream's TMEM columns
constexpr int kStages = 4;
constexpr int kRaw = 3;                                  // raw stages of 8-bit codes
constexpr int kQBytes = kTileRows * kKvHeadDim * 2;
constexpr int kTileBytes = kStageKeys * kKvHeadDim * 2;  // a K or V tile: 16 KB
constexpr int kOutPitch = 68;                            // floats of a row of O in shared memory
constexpr float kNone = -1e30f;  // reference of a row without a score yet: any finite score overflows it
constexpr float kMostSum = 512.f;  // of a row's weights in a unit, before its reference moves

constexpr int kColFloats = 8 * 20;                        // of a stage's K or V factors, see col_at

struct TcSmem {
  static constexpr int kQ = 0;                                   // 2 Q tiles
  static constexpr int kKV = kQ + 2 * kQBytes;                   // stages of K, V
  static constexpr int kRawOff = kKV + kStages * 2 * kTileBytes; // raw stages of K, V codes
  static constexpr int kRawScale = kRawOff + kRaw * kTileBytes;  // [raw stage][2][128]
  static constexpr int kCol = kRawScale + kRaw * 2 * kStageKeys * 4;  // [stage][2][128]: K, V factors, see col_at
  static constexpr int kBars = kCol + kStages * 2 * kColFloats * 4;
  static constexpr int kNumBars = 2 * kStages + 2 * 3 * kBufs + 2 * 2 + 1;
  static constexpr int kStat = (kBars + kNumBars * 8 + 15) / 16 * 16;  // [stream][128] (ref, sum), after the loop
  static constexpr int kMisc = kStat + 2 * kTileRows * 8;
  static constexpr int kTotal = kMisc + 16 + 1024;               // + alignment slack
  static_assert(2 * kTileRows * kOutPitch * 4 <= kRawOff - kKV, "the streams' outputs fit the stages");
  static_assert(kTotal <= 232448, "shared memory of a CTA");
};

__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 16 TMEM lanes x 8·N columns: thread t has, for each group c of 8 columns, lane t/4 columns 8c + 2(t%4) + {0, 1}
// in r[4c], r[4c+1] and the same of lane t/4 + 8 in r[4c+2], r[4c+3].
__device__ __forceinline__ void tmem_ld_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_x2(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_x2(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 lanes x 32 columns of 16-bit pairs: r[2c] is lane t/4, column 4c + t%4; r[2c+1] lane t/4 + 8.
__device__ __forceinline__ void tmem_st_pairs(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Waits for this thread's tcgen05.ld; the registers pass through so that no use moves above it.
template <int N>
__device__ __forceinline__ void tmem_ld_wait_regs(uint32_t (&r)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

// One thread of the warp. MMAs are issued from warp-uniform code under it: under a branch on the lane id their
// operands are not known to be uniform, and each issue takes some 130 cycles.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float lds_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts_u4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void sts_f(uint32_t addr, float x) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}

// Pairs of fp32 in one instruction (64-bit registers).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return d;
}

// mbar_wait that pauses for NS nanoseconds between polls: the loaders and issuers wait most of the time, and with
// plain polls (one in 40 cycles, whatever suspend time is asked for) half of all instructions were theirs.
template <int NS>
__device__ __forceinline__ bool mbar_wait_paused(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                 uint32_t* status, uint32_t code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = sm_cycles();
  for (;;) {
    __nanosleep(NS);
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (sm_cycles() - t0 > kWaitBudgetCycles) break;
  }
  *abort_flag = 1;
  atomicCAS(status, 0u, code);
  return false;
}

// Registers of the calling warpgroup's threads. The block is launched with 128 a thread (4 warpgroups, 512);
// 88 (loaders) + 2 x 192 (softmax) + 40 (issuers) are the same 512.
template <int N>
__device__ __forceinline__ void regs_less() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_more() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// N bytes to shared memory by cp.async; zeros where !live.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t saddr, const void* g, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(g), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_or_zero(uint32_t saddr, const void* g, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(saddr), "l"(g), "r"(live ? 4 : 0) : "memory");
}

// A value's scale as 2^e (for the widened code) and the factor left for its weight. e is kept where code·2^e is
// in the type's range; a non-finite scale stays in the factor.
template <typename T>
__device__ __forceinline__ float scale_power(float y) {
  const float p = __uint_as_float(__float_as_uint(y) & 0x7f800000u);
  constexpr float lo = std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-110f;
  constexpr float hi = std::is_same<T, __half>::value ? 0x1p7f : 0x1p110f;
  return fminf(fmaxf(p, lo), hi);
}

template <typename T>
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  const auto r = __hmul2(*reinterpret_cast<typename H2<T>::V*>(&a), *reinterpret_cast<typename H2<T>::V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Place of key j's factors in a stage: the 16 keys of a unit that a softmax thread sees (8c + 2t + {0, 1}) lie
// together, the four threads' blocks a quarter of the banks apart.
constexpr int kColPitch = 20;
__device__ __forceinline__ int col_at(int j) {
  return ((j >> 6) * 4 + ((j >> 1) & 3)) * kColPitch + ((j >> 3) & 7) * 2 + (j & 1);
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kTcThreads, 1) attn_prefix_tc_kernel(PrefixArgs a, uint32_t* status) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool Q8 = KIND != B2P_KV_16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_col = reinterpret_cast<float*>(smem + TcSmem::kCol);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + TcSmem::kBars);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* s_full = kv_empty + kStages;    // [stream][buffer], as the next two
  uint64_t* p_full = s_full + 2 * kBufs;
  uint64_t* o_full = p_full + 2 * kBufs;    // O with the buffer's unit in it
  uint64_t* drain = o_full + 2 * kBufs;     // [stream][issuer]
  uint64_t* q_full = drain + 4;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + TcSmem::kMisc);
  volatile uint32_t* abort_flag = tmem_holder + 1;

  // (shuffled, so that what follows from them is known to be uniform: TMEM addresses have to be)
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kvh = blockIdx.y;
  // this CTA's row tiles (one, or two from an even number) and keys
  const int pairs = a.pair_rows / (2 * kTileRows);
  const bool two = (int)blockIdx.x < pairs * a.n_prefix;
  const int part = two ? (int)blockIdx.x / pairs : (int)blockIdx.x - pairs * a.n_prefix;
  const int row_base = two ? ((int)blockIdx.x % pairs) * 2 * kTileRows : a.pair_rows;
  const int chunk = two ? a.prefix_chunk : a.last_chunk;
  const int first = part * chunk;
  const int nkeys = min(a.prefix_len - first, chunk);
  const int stages = (nkeys + kStageKeys - 1) / kStageKeys;
  const int units = (nkeys + kUnitKeys - 1) / kUnitKeys;
  // stream s: row tile s and every unit of keys, or units s, s + 2, ... of the one row tile
  auto units_of = [&](int s) { return two ? units : (units - s + 1) / 2; };
  auto unit_of = [&](int s, int i) { return two ? i : 2 * i + s; };  // (two to a stage)

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&kv_full[i], 4);
      mbar_init(&kv_empty[i], 2);
    }
    for (int i = 0; i < 2 * kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&drain[i], 1);
    mbar_init(q_full, 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kIssueWarp0) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, *tmem_holder, 0);
  // Inputs are complete from here on; only then may the next kernel start, so that it need not wait for this one
  // before it reads the same inputs.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp < kSoftWarp0) {
    // ---------------- load and widen ----------------
    regs_less<88>();
    const int tid = threadIdx.x;
    const int sh = a.c.page_shift, mask = (1 << sh) - 1;
    const uint32_t kv_base = smem_u32(smem + TcSmem::kKV);
    const uint32_t raw_base = smem_u32(smem + TcSmem::kRawOff);
    const uint32_t scale_base = smem_u32(smem + TcSmem::kRawScale);
    // Pages of four keys `step` apart, as the list has them; then, when they have arrived, negative past the part's end or
    // where the list is wrong. And a key's vector index in its page.
    struct Pages {
      int of[4];
    };
    auto pages = [&](int key, int step) {
      Pages p;
#pragma unroll
      for (int i = 0; i < 4; ++i) p.of[i] = a.prefix_pages[(first + min(key + i * step, nkeys - 1)) >> sh];
      return p;
    };
    auto checked = [&](Pages p, int key, int step) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool bad = (unsigned)p.of[i] >= (unsigned)a.c.n_pages;
        if (bad) atomicCAS(status, 0u, (uint32_t)DEV_BAD_ARGS);
        if (bad || key + i * step >= nkeys) p.of[i] = -1;
      }
      return p;
    };
    auto vec_at = [&](int page, int key) { return a.c.vec(max(page, 0), kvh, (first + key) & mask); };
    if constexpr (Q8) {
      // one cp.async group a stage; a thread widens the pieces that it loaded itself
      auto stage_pages = [&](int n) { return pages(n * kStageKeys + (tid >> 2), 32); };
      // Of each of its four keys a thread loads 16 codes of K and V, and the first of the four threads the scales.
      auto load = [&](int n, const Pages& ids) {
        const Pages p = checked(ids, n * kStageKeys + (tid >> 2), 32);
        const uint32_t raw = raw_base + (n % kRaw) * kTileBytes;
        const uint32_t sc = scale_base + ((n % kRaw) * 2 * kStageKeys + (tid >> 2)) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long at = vec_at(p.of[i], n * kStageKeys + i * 32 + (tid >> 2));
          const long long off = at * 64 + (tid & 3) * 16;
          const uint32_t dst = raw + (i * 128 + tid) * 16;
          cp_async16_or_zero(dst, a.c.k + off, p.of[i] >= 0);
          cp_async16_or_zero(dst + kTileBytes / 2, a.c.v + off, p.of[i] >= 0);
          if ((tid & 3) == 0) {
            cp_async4_or_zero(sc + i * 128, a.c.k_scale + at, p.of[i] >= 0);
            cp_async4_or_zero(sc + i * 128 + kStageKeys * 4, a.c.v_scale + at, p.of[i] >= 0);
          }
        }
        cp_async_commit();
      };
      {
        const Pages p0 = stage_pages(0), p1 = stage_pages(1), p2 = stage_pages(2);  // (past the end: zeros)
        load(0, p0);
        load(1, p1);
        load(2, p2);
      }
      for (int n = 0; n < stages; ++n) {
        const Pages next = stage_pages(n + kRaw);  // (the page ids arrive meanwhile)
        const int st = n % kStages;
        if (!__all_sync(~0u, mbar_wait_paused<500>(&kv_empty[st], ((n / kStages) & 1) ^ 1u, abort_flag, status,
                                        DEV_TIMEOUT_PRODUCER)))
          break;
        cp_async_wait<kRaw - 1>();
        __syncwarp();  // the scales come from the warp's other threads
        const uint32_t raw = raw_base + (n % kRaw) * kTileBytes + tid * 16;
        const uint32_t sc = scale_base + ((n % kRaw) * 2 * kStageKeys + (tid >> 2)) * 4;
        const uint32_t col = smem_u32(s_col) + st * 2 * kColFloats * 4;
        uint4 x[2][4];
        float scale[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            x[v][i] = lds_u4(raw + v * (kTileBytes / 2) + i * 128 * 16);
            scale[v][i] = lds_f(sc + (v * kStageKeys + i * 32) * 4);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = i * 32 + (tid >> 2);
          const float power = scale_power<T>(scale[1][i]);
          const uint32_t pw = pack_h2<T>(power, power);
          if ((tid & 3) == 0) {
            // (a score past the end is -inf)
            sts_f(col + col_at(row) * 4, n * kStageKeys + row < nkeys ? scale[0][i] * kScaleLog2 : 1.f);
            sts_f(col + (kColFloats + col_at(row)) * 4, scale[1][i] / power);
          }
          const uint32_t t = kv_base + st * 2 * kTileBytes + row * 128;
          const uint32_t c0 = ((2 * (tid & 3)) ^ (row & 7)) << 4;  // the two 16-byte chunks of the row, swizzled
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            uint32_t y[8];
            widen4<T, KIND>(x[v][i].x, y[0], y[1]);
            widen4<T, KIND>(x[v][i].y, y[2], y[3]);
            widen4<T, KIND>(x[v][i].z, y[4], y[5]);
            widen4<T, KIND>(x[v][i].w, y[6], y[7]);
            if (v) {
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = mul_h2<T>(y[e], pw);
            }
            sts_u4(t + v * kTileBytes + c0, y[0], y[1], y[2], y[3]);
            sts_u4(t + v * kTileBytes + (c0 ^ 16), y[4], y[5], y[6], y[7]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[st]);
        load(n + kRaw, next);
      }
    } else {
      bool ok = true;
      for (int n = 0; n <= stages; ++n) {
        if (n < stages) {
          const int st = n % kStages;
          ok = __all_sync(~0u, mbar_wait_paused<500>(&kv_empty[st], ((n / kStages) & 1) ^ 1u, abort_flag, status,
                                          DEV_TIMEOUT_PRODUCER));
          if (!ok) break;
          const uint32_t kt = kv_base + st * 2 * kTileBytes;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = n * kStageKeys + h * 64 + (tid >> 3);
            const Pages p = checked(pages(key, 16), key, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = (h * 4 + i) * 16 + (tid >> 3), ch = tid & 7;
              const long long off = vec_at(p.of[i], n * kStageKeys + row) * 128 + ch * 16;
              cp_async16_or_zero(kt + swz(row, ch), a.c.k + off, p.of[i] >= 0);
              cp_async16_or_zero(kt + kTileBytes + swz(row, ch), a.c.v + off, p.of[i] >= 0);
            }
          }
        }
        cp_async_commit();
        if (n > 0) {  // stage n - 1 has landed
          cp_async_wait<1>();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[(n - 1) % kStages]);
        }
      }
    }
    cp_async_wait<0>();
  } else if (warp < kIssueWarp0) {
    // ---------------- softmax: stream s, lane quarter ----------------
    regs_more<192>();
    const int s = (warp - kSoftWarp0) >> 2, quarter = warp & 3, t = lane & 3;
    const int count = units_of(s);
    const int row0 = row_base + (two ? s : 0) * kTileRows;
    const bool upper = a.rows - row0 > 64;  // (rows of this warp: 4 (0..31) + quarter)
    const uint32_t t0 = tmem + s * 256 + ((uint32_t)(quarter * 32) << 16);
    constexpr uint32_t kHalf = 16u << 16;  // from the lower 16 lanes of the quarter to the upper
    // Q tiles: row r of a tile is 128 contiguous bytes of q, and lane 32 (r % 4) + r / 4
    for (int i = threadIdx.x - kSoftWarp0 * 32; i < (two ? 2 : 1) * kTileRows * 8; i += 256) {
      const int row = i >> 3, ch = i & 7;
      const unsigned r = row_base + row, token = r / (unsigned)a.group;
      const bool live = (int)r < a.rows;
      const T* src = static_cast<const T*>(a.q);
      if (live) src += (long long)token * a.ld_q + (kvh * a.group + (r - token * a.group)) * kKvHeadDim + ch * 8;
      cp_async16_or_zero(smem_u32(smem + TcSmem::kQ) + (row >> 7) * kQBytes +
                             swz((row & 3) * 32 + ((row & 127) >> 2), ch),
                         src, live);
    }
    cp_async_commit();
    cp_async_wait<0>();
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    const uint32_t col0 = smem_u32(s_col) + t * kColPitch * 4;
    // a thread's rows: lane/4 + 8e of each half h, index 2h + e
    float2 l[4];
    float neg[4];  // references, negated
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      l[r] = make_float2(0.f, 0.f);
      neg[r] = -kNone;
    }
    // (a wait that fails ends the launch: later ones fail at once, what is computed meanwhile is not used)
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      mbar_wait(bar, parity, abort_flag, status, DEV_TIMEOUT_EPILOGUE);
      __syncwarp();
      tc_fence_after();
    };
    // Unit i is in score buffer b, used for the time ph (from 0; kept along with i, as 3 buffers divide badly).
    auto ready = [&](int i, int b, uint32_t ph) {  // its scores, and its stage's column factors
      if (Q8 && (!two || (i & 1) == 0)) {
        const int n = unit_of(s, i) >> 1;
        mbar_wait(&kv_full[n % kStages], (n / kStages) & 1, abort_flag, status, DEV_TIMEOUT_EPILOGUE);
      }
      mbar_wait(&s_full[s * kBufs + b], ph & 1, abort_flag, status, DEV_TIMEOUT_EPILOGUE);
      __syncwarp();
      tc_fence_after();
    };
    auto publish = [&](int b) {  // the weights in buffer b
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[s * kBufs + b]);
    };
    // The factors of column groups c and c + 1.
    auto factors = [&](uint32_t from, float2 (&k)[2], int c) {
      const float4 f = lds_f4(from + 8 * c);
      k[0] = make_float2(f.x, f.y);
      k[1] = make_float2(f.z, f.w);
    };
    // All units of the stream, for both halves of the lanes (H 2) or the lower one.
    auto run = [&](auto halves) {
      constexpr int H = decltype(halves)::value;
      // Part c (32 keys) of the scores in buffer b.
      auto load = [&](int b, int c, uint32_t (&x)[H][16]) {
#pragma unroll
        for (int h = 0; h < H; ++h) tmem_ld_x4(t0 + b * kUnitKeys + c * 32 + h * kHalf, x[h]);
      };
      auto loaded = [&](uint32_t (&x)[H][16]) {
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(x[h][i])::"memory");
      };
      auto mask = [&](uint32_t (&x)[H][16], int lim) {  // keys from lim on
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (8 * c + 2 * t + e >= lim) {
#pragma unroll
              for (int h = 0; h < H; ++h) x[h][4 * c + e] = x[h][4 * c + 2 + e] = 0xff800000u;
            }
      };
      // 16-bit weights of a part, and the rows' sums.
      auto weigh = [&](const uint32_t (&x)[H][16], uint32_t col, uint32_t (&pk)[H][16], int at, float2 (&sum)[4]) {
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          float2 kc[2] = {make_float2(kScaleLog2, kScaleLog2), make_float2(kScaleLog2, kScaleLog2)}, vf[2];
          if (Q8) factors(col, kc, c), factors(col + kColFloats * 4, vf, c);
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = 2 * h + (k & 1);
              const uint32_t* v = x[h] + 4 * c + 2 * k;
              const float2 y = fma2(make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])), kc[k >> 1],
                                    make_float2(neg[r], neg[r]));
              float2 w = make_float2(exp2_sfu(y.x), exp2_sfu(y.y));
              sum[r] = add2(sum[r], w);
              if (Q8) w = mul2(w, vf[k >> 1]);
              pk[h][at + 2 * c + k] = pack_h2<T>(w.x, w.y);
            }
        }
      };
      // The rows' references go above the scores of unit i (buffer b, used for the time ph); what was summed is scaled.
      auto raise = [&](int i, int b, uint32_t ph, uint32_t col, int lim) {
        float top[2 * H];
#pragma unroll
        for (int r = 0; r < 2 * H; ++r) top[r] = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t x[H][16];
          load(b, c, x);
          loaded(x);
          mask(x, lim - 32 * c);
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            float2 kc[2] = {make_float2(kScaleLog2, kScaleLog2), make_float2(kScaleLog2, kScaleLog2)};
            if (Q8) factors(col + 32 * c, kc, g);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float2 f = kc[k >> 2];
                const int r = 2 * h + ((k >> 1) & 1);
                top[r] = fmaxf(top[r], __uint_as_float(x[h][4 * g + k]) * (k & 1 ? f.y : f.x));
              }
          }
        }
        float f[2 * H];
#pragma unroll
        for (int r = 0; r < 2 * H; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 2));
          const float now = fminf(neg[r], -ceilf(top[r]));
          f[r] = now == neg[r] ? 1.f : exp2_sfu(now - neg[r]);
          neg[r] = now;
          l[r] = mul2(l[r], make_float2(f[r], f[r]));
        }
        if (i > 0) {
          // every unit before this one is in O
          wait(&o_full[s * kBufs + (b ? b - 1 : kBufs - 1)], (b ? ph : ph - 1) & 1);
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[8];
              tmem_ld_x2(t0 + kOCol + c * 16 + h * kHalf, o);
              tmem_ld_wait_regs(o);
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f[2 * h + ((k >> 1) & 1)]);
              tmem_st_x2(t0 + kOCol + c * 16 + h * kHalf, o);
            }
        }
      };
      // A part's scores are on their way while the one before is weighed, and a unit's weights are published when
      // their stores have had the time of the next part to end. LAST: no next unit, and the keys may end in this one.
      uint32_t xa[H][16];
      auto unit = [&](auto last, int i, int b, uint32_t ph) {
        constexpr bool LAST = decltype(last)::value;
        const int u = unit_of(s, i);
        const uint32_t col = col0 + ((u >> 1) % kStages) * (2 * kColFloats * 4) + (u & 1) * (4 * kColPitch * 4);
        const int lim = LAST ? nkeys - u * kUnitKeys : kUnitKeys;  // keys left
        uint32_t xb[H][16], pk[H][16];
        float2 sum[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = make_float2(0.f, 0.f);
        loaded(xa);
        load(b, 1, xb);
        if (LAST) mask(xa, lim);
        weigh(xa, col, pk, 0, sum);
        if (i > 0) publish(b ? b - 1 : kBufs - 1);
        loaded(xb);
        if (LAST) {
          mask(xb, lim - 32);
        } else {
          const int bn = b + 1 < kBufs ? b + 1 : 0;
          ready(i + 1, bn, b + 1 < kBufs ? ph : ph + 1);
          load(bn, 0, xa);
        }
        weigh(xb, col + 32, pk, 8, sum);
        bool fits = true;
#pragma unroll
        for (int r = 0; r < 2 * H; ++r) fits = fits && sum[r].x + sum[r].y <= kMostSum;
        if (__any_sync(~0u, !fits)) {  // again, from scores that are still there
          raise(i, b, ph, col, lim);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[r] = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            load(b, c, xb);
            loaded(xb);
            if (LAST) mask(xb, lim - 32 * c);
            weigh(xb, col + 32 * c, pk, 8 * c, sum);
          }
        }
#pragma unroll
        for (int r = 0; r < 2 * H; ++r) l[r] = add2(l[r], sum[r]);
#pragma unroll
        for (int h = 0; h < H; ++h) tmem_st_pairs(t0 + b * kUnitKeys + h * kHalf, pk[h]);
        if (LAST) publish(b);
      };
      {
        const int u = unit_of(s, 0);
        raise(0, 0, 0, col0 + (u & 1) * (4 * kColPitch * 4), nkeys - u * kUnitKeys);
        load(0, 0, xa);
      }
      int b = 0;
      uint32_t ph = 0;
#pragma unroll 1
      for (int i = 0; i + 1 < count; ++i) {
        unit(std::false_type(), i, b, ph);
        if (++b == kBufs) b = 0, ++ph;
      }
      unit(std::true_type(), count - 1, b, ph);
    };
    if (count > 0) {
      ready(0, 0, 0);
      if (upper)
        run(std::integral_constant<int, 2>());
      else
        run(std::integral_constant<int, 1>());
    }
    // the streams' outputs meet in the stages' memory, once no MMA reads it any more
    if (count > 0) wait(&o_full[s * kBufs + (count - 1) % kBufs], ((count - 1) / kBufs) & 1);
    named_bar_sync(2, 256);
    float* s_o = reinterpret_cast<float*>(smem + TcSmem::kKV);
    float2* s_stat = reinterpret_cast<float2*>(smem + TcSmem::kStat);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && !upper) break;
      const int lane_row = h * 64 + 4 * (lane >> 2) + quarter;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t o[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = 0;
        if (count > 0) {
          tmem_ld_x4(t0 + kOCol + c * 32 + h * kHalf, o);
          tmem_ld_wait_regs(o);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* dst = s_o + (s * kTileRows + lane_row + e * 32) * kOutPitch + c * 32 + 2 * t;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<float2*>(dst + 8 * k) =
                make_float2(__uint_as_float(o[4 * k + 2 * e]), __uint_as_float(o[4 * k + 2 * e + 1]));
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 2 * h + e;
        float sum = l[r].x + l[r].y;
        sum += __shfl_xor_sync(~0u, sum, 1);
        sum += __shfl_xor_sync(~0u, sum, 2);
        if (t == 0)
          s_stat[s * kTileRows + lane_row + e * 32] = make_float2(neg[r] == -kNone ? -INFINITY : -neg[r], sum);
      }
    }
    named_bar_sync(2, 256);
    if (*abort_flag == 0) {
      for (int i = threadIdx.x - kSoftWarp0 * 32; i < (two ? 2 : 1) * kTileRows * 16; i += 256) {
        const int tile = i >> 11, row = (i >> 4) & 127, d = (i & 15) * 4;
        const int r = row_base + tile * kTileRows + row;
        if (r >= a.rows) continue;
        const long long at = ((long long)part * gridDim.y + kvh) * a.rows + r;
        const float2 st0 = s_stat[tile * kTileRows + row];
        float sum = st0.y, top = st0.x;
        float4 acc = *reinterpret_cast<const float4*>(s_o + (tile * kTileRows + row) * kOutPitch + d);
        if (!two) {  // both streams have these rows, each with its reference
          const float2 st1 = s_stat[kTileRows + row];
          const float4 y = *reinterpret_cast<const float4*>(s_o + (kTileRows + row) * kOutPitch + d);
          top = fmaxf(st0.x, st1.x);
          const float base = top == -INFINITY ? 0.f : top;
          const float f0 = exp2_sfu(st0.x - base), f1 = exp2_sfu(st1.x - base);
          sum = f0 * sum + f1 * st1.y;
          acc = make_float4(f0 * acc.x + f1 * y.x, f0 * acc.y + f1 * y.y, f0 * acc.z + f1 * y.z,
                            f0 * acc.w + f1 * y.w);
        }
        *reinterpret_cast<float4*>(a.part_o + at * kKvHeadDim + d) = acc;
        if (d == 0) a.part_ml[at] = make_float2(top, sum);
      }
    }
  } else {
    // ---------------- MMA issuers: scores of stream 0, 1, outputs of stream 0, 1 ----------------
    regs_less<40>();
    const int role = warp - kIssueWarp0;
    const int s = role & 1;
    const int count = units_of(s);
    const uint32_t kv_base = smem_u32(smem + TcSmem::kKV);
    const uint32_t ts = tmem + s * 256;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(~0u, mbar_wait_paused<120>(bar, parity, abort_flag, status, DEV_TIMEOUT_MMA)) != 0;
    };
    bool ok = true, issued = false;
    int b = 0;
    uint32_t ph = 0;
    if (role < 2) {
      const uint32_t idesc = umma_idesc_f16(BF16, kTileRows, kUnitKeys);
      const uint64_t q_desc = sw128_kmajor_desc(smem_u32(smem + TcSmem::kQ + (two ? s : 0) * kQBytes));
      const uint64_t kv_desc = sw128_kmajor_desc(kv_base);
      ok = wait(q_full, 0);
      for (int i = 0; ok && i < count; ++i) {
        const int u = unit_of(s, i), n = u >> 1, st = n % kStages;
        ok = wait(&kv_full[st], (n / kStages) & 1) &&
             (i < kBufs || wait(&o_full[s * kBufs + b], (ph - 1) & 1));  // the buffer's last weights are in O
        if (!ok) break;
        tc_fence_after();
        const uint64_t k_desc = kv_desc + ((st * 2 * kTileBytes + (u & 1) * kUnitKeys * 128) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kKvHeadDim / 16; ++k)
            umma_f16_ss(ts + b * kUnitKeys, q_desc + 2 * k, k_desc + 2 * k, idesc, k > 0 ? 1u : 0u);
          umma_commit(&s_full[s * kBufs + b]);
        }
        __syncwarp();
        issued = true;
        if (++b == kBufs) b = 0, ++ph;
      }
    } else {
      const uint32_t idesc = umma_idesc_f16(BF16, kTileRows, kKvHeadDim) | (1u << 16);  // B = V, MN-major
      const uint64_t kv_desc = sw128_mn_desc(kv_base + kTileBytes, 16);
      for (int i = 0; i < count; ++i) {
        const int u = unit_of(s, i), st = (u >> 1) % kStages;
        ok = wait(&p_full[s * kBufs + b], ph & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v_desc = kv_desc + ((st * 2 * kTileBytes + (u & 1) * kUnitKeys * 128) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kUnitKeys / 16; ++k)
            umma_f16_ts(ts + kOCol, ts + b * kUnitKeys + k * 8, v_desc + k * (2048 >> 4), idesc,
                        i > 0 || k > 0 ? 1u : 0u);
          umma_commit(&o_full[s * kBufs + b]);
          if (!two || (u & 1)) umma_commit(&kv_empty[st]);  // the stream's last unit of the stage
        }
        __syncwarp();
        issued = true;
        if (++b == kBufs) b = 0, ++ph;
      }
    }
    if (!ok && issued) {
      if (elect_one()) umma_commit(&drain[role]);
      __syncwarp();
      mbar_wait_drain(&drain[role], 0);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename T, int KIND>
int launch_tc(const PrefixArgs& a, cudaStream_t st) {
  DeviceCtx* c = nullptr;
  int rc = ctx_get(&c);
  if (rc) return rc;
  static thread_local uint64_t attr_mask = 0;  // one per instantiation
  if (!(attr_mask & (1ull << (c->device & 63)))) {
    B2P_CHECK_CUDA(cudaFuncSetAttribute(attn_prefix_tc_kernel<T, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        TcSmem::kTotal));
    attr_mask |= 1ull << (c->device & 63);
  }
  const long long ctas = (long long)(a.pair_rows / (2 * kTileRows)) * a.n_prefix + a.n_last;
  B2P_REQUIRE(ctas < (1ll << 31), "too much work for one call");
  B2P_CHECK_CUDA(launch_pdl(attn_prefix_tc_kernel<T, KIND>, dim3((unsigned)ctas, a.c.kv_heads), dim3(kTcThreads),
                            TcSmem::kTotal, st, a, c->status));
  B2P_POST_LAUNCH();
  return B2P_OK;
}

}  // namespace

// As many parts as leave each SM one CTA. A CTA with one row tile has half the work of one with two for the same
// keys, so the odd tile's parts are about twice as long.
void prefix_tc_plan(int rows, int kv_heads, int prefix_len, PrefixSplit* s) {
  const int tiles = ceil_div(rows, kTileRows), pairs = tiles / 2, odd = tiles & 1;
  const int stages = ceil_div(prefix_len, kStageKeys);
  *s = PrefixSplit();
  s->pair_rows = pairs * 2 * kTileRows;
  auto last = [&](int parts) { return pairs ? ceil_div(parts, 2) : parts; };
  int parts = 1;
  while (parts < stages && (long long)kv_heads * (pairs * (parts + 1) + odd * last(parts + 1)) <= kSms) ++parts;
  if (pairs) {
    s->prefix_chunk = ceil_div(stages, parts) * kStageKeys;
    s->n_prefix = ceil_div(prefix_len, s->prefix_chunk);
  }
  if (odd) {
    s->last_chunk = ceil_div(stages, last(parts)) * kStageKeys;
    s->n_last = ceil_div(prefix_len, s->last_chunk);
  }
}

int launch_prefix_tc(const PrefixArgs& a, bool bf16, cudaStream_t st) {
  switch (a.c.kind) {
    case B2P_KV_INT8:
      return bf16 ? launch_tc<__nv_bfloat16, B2P_KV_INT8>(a, st) : launch_tc<__half, B2P_KV_INT8>(a, st);
    case B2P_KV_E4M3:
      return bf16 ? launch_tc<__nv_bfloat16, B2P_KV_E4M3>(a, st) : launch_tc<__half, B2P_KV_E4M3>(a, st);
    default:
      return bf16 ? launch_tc<__nv_bfloat16, B2P_KV_16>(a, st) : launch_tc<__half, B2P_KV_16>(a, st);
  }
}

}  // namespace b2p
