// prompt.cu -- attention over whole prompts, packed sequences, on tcgen05.
//
// For sequence b of lq new tokens (rows cu_q[b] .. of the packed q) and lk
// keys (rows cu_k[b] .. of the packed k / v), query token i, head h, kv head
// h / group:
//   s_j = scale * q_i . k_j,  j <= i + lk - lq when causal (bottom-right),
//   o   = sum_j softmax(s)_j v_j,   lse = log sum_j exp(s_j)
// in one pass over the keys with a running row maximum and sum.
//
// A work item is (sequence, kv head, 2 Q tiles).  A Q tile packs the group's
// heads with its tokens: row = token * group + head, 128 / group tokens, so
// that one K / V tile read from L2 serves every head of the group and the
// causal diagonal wastes few columns.  The two Q tiles are independent streams
// of steps over key tiles of 128 that share the K / V tiles: while one tile's
// warps take exponentials, the tensor pipe computes the other's products.
//
// What bounds it.  Per Q tile and step the tensor pipe needs 2 * 128 * 128 *
// (d_qk + d_v) flops at 8192 a cycle (1024 cycles at head size 128) and the
// exponentials 128 * 128 at 16 a cycle (1024 cycles): 2048 cycles for a step of
// both tiles, were either always busy.  A tile's own chain is longer: S read
// and its maximum 600 cycles, exponentials 1400, the last value products and
// the next scores 1100, in all 3100 to 3300, and with two tiles per SM (S and O
// of a third do not fit in TMEM) that chain is the bound.  Hence two threads
// a row (shorter maxima and exponentials), P handed over as 48 + 16 of a half's
// 64 columns (most of the value product runs under the last exponentials), maxima
// exchanged only when one has to move, and O rescaled only past a factor 2^8.
//
// Measured: one causal prompt of 8192 tokens, 64 query / 8 kv heads of 128,
// bf16: 942 us for launches 20 ms apart (SM clock 1965 MHz, 1.17 PFLOP/s), 1040 us in
// a loop under the power cap (1605 MHz, 1.06 PFLOP/s); the tensor pipe is active 61% of
// the cycles, 45% of those of 16 packed prompts of 1 to 2048 tokens (451 us apart, 486 in
// a loop at 1657 MHz); 2 prompts of 1000 to 2048 tokens, 128 heads of 192 / 128: 352 and
// 378 us; 256 tokens over 16256 keys: 152 us (about 224 without split keys);
// one prompt of 37 tokens: 11.4 us.
//
//   warps 0-7 / 8-15: rows of Q tile 0 / 1 (two threads per row, S read from
//     TMEM, P written over it as the A operand of P V)
//   warp 16: MMA issuer    warp 17: TMA producer    warp 18: scheduler
//   warp 19: value rows at the edge
//
// A weight of 0 does not hide a value: 0 * NaN is NaN.  In V tiles with keys
// that not every row of the unit sees, warp 19 (with one V stage the row warps) clears
// the rows that none sees, the next sequence's among them, and every infinity or NaN
// that only some see, and notes its key; the rows that see it add it to what they store.
//
// TMEM: S0 S1 (128 columns each, P in place), O0 O1.  A tile's products are
// issued in order, so the barrier that announces S of step j also says that P V of
// step j - 1 is complete: the rows rescale O without a further wait.
//
// One rounding below 32 bits: P, to the inputs' type, as the value product's
// operand.  The row sum adds the unrounded values; S, O, maxima and
// sums are f32.
//
// Every mbarrier wait is bounded (common.cuh).
#include <algorithm>

#include "common.cuh"
#include "flagattn_b200.h"
#include "merge.cuh"

namespace fa {
namespace prompt {

// The last warpgroup gives registers to the row warps: 16 * 112 + 4 * 32 = 20 *
// 96, the launch's (launch_t refuses any other: a split with a larger sum waits for ever).
constexpr int kThreads = 640, kRowRegs = 112, kOtherRegs = 32;
constexpr int kRowWarps = 16, kMmaWarp = 16, kProducerWarp = 17, kSchedulerWarp = 18, kEdgeWarp = 19;
constexpr int kTile = 128;                 // rows of a Q tile, keys of a K / V tile
constexpr uint32_t kTmemCols = 512;
// O is rescaled only when the maximum grows by more than this (log2 units):
// P stays below 2^8, and the sum and O carry the same factor.
constexpr float kRescaleThreshold = 8.0f;

template <int kDqk, int kDv>
struct Plan {
  static constexpr int kQkChunks = kDqk / 64, kVChunks = kDv / 64;
  static constexpr int kChunkBytes = kTile * 128;  // 128 rows x 64 dims, 128-byte swizzle
  static constexpr int kQBytes = kQkChunks * kChunkBytes;   // one Q tile
  static constexpr int kKBytes = kQkChunks * kChunkBytes;
  static constexpr int kVBytes = kVChunks * kChunkBytes;
  static constexpr int kKStages = kDqk == 192 ? 2 : (kDqk == 128 ? 3 : 4);
  static constexpr int kVStages = kDqk == 192 ? 1 : (kDqk == 128 ? 2 : 4);
  // With one stage a V tile lands when its products are due: its readers' 256
  // threads clear it (a few hundred cycles) and not one warp (about 2000; 2 prompts
  // of 1000 to 2048 tokens, 128 heads of 192 / 128: 395 us so, 363 by the rows).
  static constexpr bool kRowsClear = kVStages == 1;
  static constexpr int kOffX = 1024;
  static constexpr int kOffQ = kOffX + 2048;  // past the exchange block
  static constexpr int kOffK = kOffQ + 2 * kQBytes;
  static constexpr int kOffV = kOffK + kKStages * kKBytes;
  static constexpr int kSmemUsed = kOffV + kVStages * kVBytes;
  static constexpr int kSmemBytes = kSmemUsed;
  static constexpr uint32_t kColS = 0, kColO = 2 * kTile;
  static_assert(kColO + 2 * kDv <= kTmemCols, "TMEM plan");
  static_assert(kSmemBytes <= 232448, "shared memory plan exceeds 227 KB");
};

// One unit of work, as the scheduler warp hands it to the others.  Key tiles
// [j0, j1); Q tile x takes those below end[x].
struct Work {
  int kvh;                 // -1: no more work
  int q0, lq, k0, lk, i0;  // i0: first token of Q tile 0 in its sequence
  int j0, j1, end[2];
  int split;
};

struct Bars {
  uint64_t q_full[2], q_empty[2];  // per Q tile
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t v_raw[4];               // a V tile that the edge warp has to look at first
  uint64_t s_full[2], o_full[2];
  uint64_t p_full[2][2];  // [Q tile][first 48 / last 16 columns of both halves]
  uint64_t work_full[2], work_empty[2];
  uint64_t cancel_full;
  uint64_t drain;
  uint4 cancelled;  // response of the launch control unit
  Work work[2];
  uint32_t tmem_base;
  int abort_flag;
  // Keys of unit k whose infinities or NaN were cleared, from the unit's first
  // hidden key on, in marks[k % 3]: a unit is handed out when all warps have begun
  // the last but one, so three are told apart.
  struct Marks {
    uint32_t any, keys[8];
  } marks[3];
};
// Row maxima, at the end row sums, that the two threads of a row exchange.
struct Exchange {
  float v[2][2][kTile];  // [Q tile][half][row]
};
static_assert(sizeof(Exchange) == 2048, "exchange block");
static_assert(sizeof(Bars) <= 1024, "barrier block");

struct Params {
  const int32_t *cu_q, *cu_k;
  const void *v;  // as the tensor map has it
  int64_t v_st, v_sh;
  int32_t batch, total_q, total_k, hq, hkv, group, tq;  // tq: tokens of a Q tile
  int32_t items;     // upper bound of the (sequence, Q tile pair) items
  int32_t splits;    // units an item's keys are cut into
  int32_t section;   // kv heads whose units go together
  int32_t d_v, causal;
  float scale_log2;
  void *o;
  int64_t o_st, o_sh;
  float *lse;  // nullable, [hq][total_q]
  float *part_o, *part_lse;  // splits > 1: [split][hq][total_q] ([d_v])
  int *status;
};

// Rows [start, end) of sequence b in a packed tensor of `total` rows; offsets
// outside it or out of order are cut to what exists.
__device__ __forceinline__ void seq_range(const int32_t *cu, int b, int total, int &start,
                                          int &len) {
  start = min(max(__ldg(cu + b), 0), total);
  len = min(max(__ldg(cu + b + 1), start), total) - start;
}

// Keys that every row, and that any row of a unit sees: [0, all), [0, some).
struct Seen {
  int all, some;
};
__device__ __forceinline__ Seen seen_keys(const Params &p, const Work &w) {
  if (!p.causal) return {w.lk, w.lk};
  const int last = min(w.i0 + 2 * p.tq, w.lq);  // past the last token
  return {max(w.i0 + 1 + w.lk - w.lq, 0), max(last + w.lk - w.lq, 0)};
}

// mbar_wait without its out-of-line loop: setmaxnreg does not go with calls.
__device__ __forceinline__ bool wait_inline(uint32_t bar, uint32_t parity, volatile int *abort_flag,
                                            int *status, int code) {
  if (mbar_test(bar, parity)) return true;
  const long long t0 = clock64();
#pragma unroll 1
  for (uint32_t i = 1;; ++i) {
    if (mbar_test(bar, parity)) return true;
    if ((i & 63u) == 0) {
      if (*abort_flag) return false;
      if (clock64() - t0 > kWaitLimitCycles) {
        *abort_flag = 1;
        if (status) atomicExch(status, code);
        return false;
      }
    }
  }
}
// Warp-wide bounded wait: all lanes return the same verdict.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag,
                                          int *status, int code) {
  return __all_sync(0xffffffffu, wait_inline(bar, parity, abort_flag, status, code)) != 0;
}
template <int kRegs>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Named barrier that returns whether any of its threads' predicates holds.
__device__ __forceinline__ bool barrier_any(int id, int threads, bool pred) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(pred))
      : "memory");
  return any != 0;
}
// Maximum that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 0 * x + y of two halves.
template <typename T>
__device__ __forceinline__ uint32_t zero_of(uint32_t x, uint32_t y) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value)
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0u), "r"(y));
  else
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0u), "r"(y));
  return d;
}

// Clears what rows of a V tile may hold that its readers must not meet: rows r0 ..
// r1 - 1 lose infinities and NaN, which are noted (key0: the tile's first key, from
// the unit's first hidden one on), rows from r1 on everything.  Done by n threads, i
// of which calls; 16-byte units, kLoads on their way at a time.
template <typename T, int kChunks, int kChunkBytes, int kLoads>
__device__ __forceinline__ void clear_hidden(uint8_t *tile, int r0, int r1, int key0,
                                             Bars::Marks &marks, int i, int n) {
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  auto finite = [](uint32_t y) {  // its halves, 0 for an infinity or a NaN
    if ((y & 0x7fffu) >= kInf) y &= 0xffff0000u;
    if ((y >> 16 & 0x7fffu) >= kInf) y &= 0xffffu;
    return y;
  };
#pragma unroll
  for (int ch = 0; ch < kChunks; ++ch) {
    uint4 *at = reinterpret_cast<uint4 *>(tile + ch * kChunkBytes);
    for (int u0 = r0 * 8 + i; u0 < r1 * 8; u0 += n * kLoads) {
      uint4 x[kLoads];
      uint32_t none = 0u;  // 0 * x + 0 is 0 unless x is an infinity or a NaN
#pragma unroll
      for (int k = 0; k < kLoads; ++k) x[k] = at[min(u0 + n * k, r1 * 8 - 1)];
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        none |= zero_of<T>(x[k].x, zero_of<T>(x[k].y, zero_of<T>(x[k].z, zero_of<T>(x[k].w, 0u))));
      if (none == 0u) continue;
#pragma unroll 1
      for (int k = 0; k < kLoads && u0 + n * k < r1 * 8; ++k) {
        const int u = u0 + n * k;
        const uint4 y = at[u], z = make_uint4(finite(y.x), finite(y.y), finite(y.z), finite(y.w));
        if (((y.x ^ z.x) | (y.y ^ z.y) | (y.z ^ z.z) | (y.w ^ z.w)) == 0u) continue;
        const int key = key0 + u / 8;  // fewer than a unit's tokens
        atomicOr(&marks.keys[key >> 5], 1u << (key & 31));
        atomicOr(&marks.any, 1u);
        __threadfence_block();  // who finds the element cleared finds its mark
        at[u] = z;
      }
    }
#pragma unroll 4
    for (int u = r1 * 8 + i; u < kTile * 8; u += n) at[u] = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
}

// Rows of Q tile x: two threads per row, each with half of the key tile's
// columns (`half`) and of O's.  A wait that gives up does not end the loop
// (every wait returns at once from then on): the two warps of a row keep
// meeting at their named barrier.
template <typename T, int kDqk, int kDv>
__device__ __forceinline__ void row_role(const Params &p, const Work &it, Bars *bars,
                                         uint8_t *smem, uint32_t tmem, int warp, int lane,
                                         uint32_t &steps, uint32_t &outs, uint32_t unit,
                                         uint32_t tiles) {
  using PL = Plan<kDqk, kDv>;
  constexpr int kCols = kTile / 2, kOCols = kDv / 2;
  volatile int *abort_flag = &bars->abort_flag;
  const int x = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
  const int row = quad * 32 + lane;
  const int tok = it.i0 + x * p.tq + row / p.group;  // token in its sequence
  const int head = it.kvh * p.group + row % p.group;
  const bool live = row < p.tq * p.group && tok < it.lq;
  const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
  // this half's S columns; its P (32 words) goes over the first of them
  const uint32_t t_s = tmem + lane_off + PL::kColS + x * kTile + half * kCols;
  const uint32_t t_o = tmem + lane_off + PL::kColO + x * kDv + half * kOCols;
  float *mine = reinterpret_cast<Exchange *>(smem + PL::kOffX)->v[x][half] + row;
  volatile float *other = reinterpret_cast<Exchange *>(smem + PL::kOffX)->v[x][half ^ 1] + row;
  const int meet = 1 + x * 4 + quad;  // named barrier of the row's two warps
  // keys this row sees: [0, end); rows without a token count as unmasked
  // (their P and O rows are never read)
  const int end = !live ? INT32_MAX
                        : (p.causal ? min(it.lk, tok + it.lk - it.lq + 1) : it.lk);
  const int n = it.end[x];
  float m_use = -INFINITY, l = 0.f;
  const uint64_t c2 = f32x2(p.scale_log2, p.scale_log2);
  for (int j = it.j0; j < n; ++j, ++steps) {
    warp_wait(smem_u32(&bars->s_full[x]), steps & 1u, abort_flag, p.status, kDevTimeoutSoftmax);
    tc_fence_after();
    float s[32], s2[32];
    tmem_ld32(t_s, s);
    tmem_ld32(t_s + 32, s2);
    const int hi = end - j * kTile - half * kCols;
    const bool masked = !__all_sync(0xffffffffu, hi >= kCols);
    tmem_wait_ld();
    if (masked) {
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        s[c] = c < hi ? s[c] : -INFINITY;  // select: whatever a masked key holds
        s2[c] = c + 32 < hi ? s2[c] : -INFINITY;
      }
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      mx[0] = max3_nan(mx[0], s[c], s[c + 1]);
      mx[1] = max3_nan(mx[1], s[c + 2], s[c + 3]);
      mx[2] = max3_nan(mx[2], s2[c], s2[c + 1]);
      mx[3] = max3_nan(mx[3], s2[c + 2], s2[c + 3]);
    }
    float m_row = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
    // a NaN score, or an infinite one, makes the row NaN
    if (!(m_row < INFINITY)) l = NAN;
    // The two halves of a row share one maximum.  It is exchanged through
    // shared memory only when some row of the two warps needs a new one; the
    // barrier itself tells.
    if (barrier_any(meet, 64, j == it.j0 || m_row * p.scale_log2 > m_use + kRescaleThreshold)) {
      *mine = m_row;
      named_bar_sync(meet, 64);
      m_row = max3_nan(m_row, *other, *other);
      named_bar_sync(meet, 64);  // read before the next exchange writes
      const float m_tile = m_row * p.scale_log2;
      bool resc = false;
      float alpha = 1.f;
      if (j == it.j0) {
        m_use = m_tile;
      } else if (m_tile > m_use + kRescaleThreshold) {
        resc = m_use != -INFINITY;  // O is all zeros while no key was visible
        alpha = resc ? fast_exp2(m_use - m_tile) : 0.f;
        l *= alpha;
        m_use = m_tile;
      }
      if (__any_sync(0xffffffffu, resc)) {
        const float a = resc ? alpha : 1.f;
#pragma unroll 1
        for (int c = 0; c < kOCols / 16; ++c) {
          float v[16];
          uint32_t u[16];
          tmem_ld16(t_o + 16 * c, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[i] * a);
          tmem_st16(t_o + 16 * c, u);
        }
      }
    }
    const float msafe = m_use == -INFINITY ? 0.f : m_use;
    const uint64_t nm2 = f32x2(-msafe, -msafe);
    uint64_t acc2 = f32x2(0.f, 0.f), acc2b = f32x2(0.f, 0.f);
    // P over S in place, 32 columns at a time
    // 16 columns of v to 8 words of w
    auto exps = [&](const float *v, uint32_t *w) {
      uint64_t y[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float x0, x1;
        f32x2_split(ffma2(f32x2(v[2 * c], v[2 * c + 1]), c2, nm2), x0, x1);
        y[c] = f32x2(fast_exp2(x0), fast_exp2(x1));
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float p0, p1;
        f32x2_split(y[c], p0, p1);
        w[c] = Elem<T>::pack2(p0, p1);
        if (c & 1)
          acc2b = fadd2(acc2b, y[c]);
        else
          acc2 = fadd2(acc2, y[c]);
      }
    };
    // P of the first 48 or the last 16 columns (and the rescaled O) is there: most of the value product runs while the last are computed
    auto hand_over = [&](int part) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars->p_full[x][part]));
    };
    uint32_t w[16], w2[16];
    exps(s, w);
    exps(s + 16, w + 8);
    tmem_st16p(t_s, w);
    exps(s2, w2);
    tmem_st8p(t_s + 16, w2);
    if constexpr (PL::kRowsClear) {
      const Seen seen = seen_keys(p, it);
      if ((j + 1) * kTile > seen.all) {  // each Q tile's warps, the first to come clears
        warp_wait(smem_u32(&bars->v_full[0]), (tiles + (j - it.j0)) & 1u, abort_flag, p.status,
                  kDevTimeoutSoftmax);
        const int r0 = max(seen.all - j * kTile, 0), r1 = min(max(seen.some - j * kTile, r0), kTile);
        clear_hidden<T, PL::kVChunks, PL::kChunkBytes, 4>(smem + PL::kOffV, r0, r1,
                                                          j * kTile - seen.all,
                                                          bars->marks[unit % 3],
                                                          (warp & 7) * 32 + lane, 256);
      }
    }
    hand_over(0);
    exps(s2 + 16, w2 + 8);
    tmem_st8p(t_s + 24, w2 + 8);
    hand_over(1);
    float a0, a1;
    f32x2_split(fadd2(acc2, acc2b), a0, a1);
    l += a0 + a1;
  }
  const bool any = n > it.j0;
  if (any) {
    *mine = l;
    named_bar_sync(meet, 64);
    l += *other;
    warp_wait(smem_u32(&bars->o_full[x]), outs & 1u, abort_flag, p.status, kDevTimeoutSoftmax);
    ++outs;
    tc_fence_after();
  }
  const float f = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
  const float lse = l == 0.f ? -INFINITY : (m_use + __log2f(l)) * 0.6931471805599453f;
  const int col0 = half * kOCols;
  // rows of the output, or (f32) of this split's partial result
  const int64_t prow = (static_cast<int64_t>(it.split) * p.hq + head) * p.total_q + it.q0 + tok;
  T *orow = static_cast<T *>(p.o) + static_cast<int64_t>(it.q0 + tok) * p.o_st + head * p.o_sh + col0;
  float *po = p.part_o + prow * p.d_v + col0;
  const Bars::Marks &marks = bars->marks[unit % 3];
  const bool marked = any && *const_cast<const volatile uint32_t *>(&marks.any) != 0;
#pragma unroll 1
  for (int c = 0; c < kOCols / 16; ++c) {
    float v[16];
    if (any) {
      tmem_ld16(t_o + 16 * c, v);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= f;
    if (marked) {
      // the cleared values of keys that this row sees: an infinity, or a NaN
      const int first = seen_keys(p, it).all;
#pragma unroll 1
      for (int key = 0; key < min(end - first, 256); ++key) {
        if (!(const_cast<const volatile uint32_t *>(marks.keys)[key >> 5] >> (key & 31) & 1u)) {
          continue;
        }
        const T *src = static_cast<const T *>(p.v) +
                       static_cast<int64_t>(it.k0 + first + key) * p.v_st + it.kvh * p.v_sh + col0 +
                       16 * c;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (col0 + 16 * c + (i & 8) >= p.d_v) break;
          const float x = Elem<T>::to_f(src[i]);
          v[i] += fabsf(x) < INFINITY ? 0.f : x;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (col0 + 16 * c + 8 * i >= p.d_v) continue;
      if (p.splits == 1) {
        uint4 u;
        u.x = Elem<T>::pack2(v[8 * i], v[8 * i + 1]);
        u.y = Elem<T>::pack2(v[8 * i + 2], v[8 * i + 3]);
        u.z = Elem<T>::pack2(v[8 * i + 4], v[8 * i + 5]);
        u.w = Elem<T>::pack2(v[8 * i + 6], v[8 * i + 7]);
        *reinterpret_cast<uint4 *>(orow + 16 * c + 8 * i) = u;
      } else {
        float4 *dst = reinterpret_cast<float4 *>(po + 16 * c + 8 * i);
        dst[0] = make_float4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3]);
        dst[1] = make_float4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]);
      }
    }
  }
  if (half == 0 && live) {
    if (p.splits > 1)
      p.part_lse[prow] = l == l ? lse : INFINITY;  // the merge's maximum would drop a NaN
    else if (p.lse)
      p.lse[static_cast<int64_t>(head) * p.total_q + it.q0 + tok] = lse;
  }
  // the O reads above precede the next unit's first product into it (issued
  // after this warp's next hand-over)
  tc_fence_before();
}

// --------------------------------------------------------------- scheduling
// The grid holds one CTA per unit; those that run take the units of CTAs not
// yet launched (cluster launch control), so every unit starts as soon as an
// SM is free for it and a CTA's set-up is paid once per SM.
__device__ __forceinline__ void cancel_next(uint32_t response, uint32_t bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], "
      "[%1];" ::"r"(response),
      "r"(bar)
      : "memory");
}
// The unit taken over (its block index), or -1 when none was left.
__device__ __forceinline__ int cancelled_block(uint32_t response) {
  uint32_t ok, x = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, h;\n\t}"
      : "=r"(ok), "=r"(x)
      : "r"(response)
      : "memory");
  return ok ? static_cast<int>(x) : -1;
}

// Finds the sequence and Q-tile pair of an item.  One warp; remembers where it
// was, since the items a CTA takes come in increasing order.
//
// Up to 32 sequences: all items by falling number of key tiles, so that the
// units that run last are short.  A lane keeps one sequence; the pairs with at
// least c key tiles are its last ones, counted in closed form, and c falls as
// the item number grows.  More sequences: sequence by sequence, each from its
// last pair (under a causal mask the one with most keys) to its first.
struct Finder {
  const Params &p;
  const int lane, span;
  int q0 = 0, k0 = 0, lq = 0, lk = 0, pairs = 0;  // of the lane's sequence
  int c = -1;                     // key tiles of the current items
  int base = 0, first = 0;        // items before them / before sequence `first`

  __device__ __forceinline__ Finder(const Params &p_, int lane_) : p(p_), lane(lane_), span(2 * p_.tq) {
    if (p.batch > 32) return;
    if (lane < p.batch) {
      seq_range(p.cu_q, lane, p.total_q, q0, lq);
      seq_range(p.cu_k, lane, p.total_k, k0, lk);
      pairs = (lq + span - 1) / span;
    }
    restart();
  }
  __device__ __forceinline__ void restart() {
    base = 0;
    c = __reduce_max_sync(0xffffffffu, pairs > 0 ? (lk + kTile - 1) / kTile : 0);
  }
  // pairs of the lane's sequence with at least n key tiles: pair i sees
  // min((i + 1) * span, lq) + lk - lq keys when causal, lk otherwise
  __device__ __forceinline__ int at_least(int n) const {
    if (n <= 0) return pairs;
    const int64_t need = static_cast<int64_t>(n - 1) * kTile + 1;
    if (!p.causal) return lk >= need ? pairs : 0;
    const int64_t t = need - lk + lq;  // tokens the pair must reach
    if (t > lq) return 0;
    const int skip = t > span ? static_cast<int>((t + span - 1) / span) - 1 : 0;
    return pairs - min(skip, pairs - 1);
  }
  __device__ __forceinline__ int inclusive_scan(int v) const {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  }
  __device__ __forceinline__ bool by_cost(int x, Work &w, int &pair) {
    if (x < base) restart();
    for (; c >= 0; --c) {
      const int more = at_least(c + 1), mine = (pairs > 0 ? at_least(c) : 0) - (pairs > 0 ? more : 0);
      const int incl = inclusive_scan(mine);
      const int all = __shfl_sync(0xffffffffu, incl, 31);
      if (x < base + all) {
        const int at = __ffs(__ballot_sync(0xffffffffu, x < base + incl)) - 1;
        pair = __shfl_sync(0xffffffffu, pairs - more - 1 + (incl - mine), at) - (x - base);
        w.q0 = __shfl_sync(0xffffffffu, q0, at);
        w.lq = __shfl_sync(0xffffffffu, lq, at);
        w.k0 = __shfl_sync(0xffffffffu, k0, at);
        w.lk = __shfl_sync(0xffffffffu, lk, at);
        return true;
      }
      base += all;
    }
    return false;  // the bound of the items is not tight
  }
  __device__ __forceinline__ bool in_order(int x, Work &w, int &pair) {
    if (x < base) base = first = 0;
    for (; first < p.batch; first += 32) {
      int s, n = 0;
      if (first + lane < p.batch) seq_range(p.cu_q, first + lane, p.total_q, s, n);
      const int incl = inclusive_scan((n + span - 1) / span);
      const int all = __shfl_sync(0xffffffffu, incl, 31);
      if (x < base + all) {
        const int at = __ffs(__ballot_sync(0xffffffffu, x < base + incl)) - 1;
        pair = base + __shfl_sync(0xffffffffu, incl, at) - 1 - x;
        seq_range(p.cu_q, first + at, p.total_q, w.q0, w.lq);
        seq_range(p.cu_k, first + at, p.total_k, w.k0, w.lk);
        return true;
      }
      base += all;
    }
    return false;
  }
  __device__ __forceinline__ bool find(int x, Work &w, int &pair) {
    return p.batch <= 32 ? by_cost(x, w, pair) : in_order(x, w, pair);
  }
};

__device__ __forceinline__ void scheduler_role(const Params &p, Bars *bars, int lane) {
  volatile int *abort_flag = &bars->abort_flag;
  const uint32_t response = smem_u32(&bars->cancelled);
  Finder finder(p, lane);
  uint32_t count = 0;  // units handed out
  int idx = blockIdx.x;
  for (uint32_t asked = 0; idx >= 0; ++asked) {
    if (lane == 0) cancel_next(response, smem_u32(&bars->cancel_full));
    // units of a section of kv heads: item by item, its splits, its heads
    const int per_section = p.items * p.splits * p.section;
    const int sec = idx / per_section, in = idx - sec * per_section;
    const int width = min(p.section, p.hkv - sec * p.section);
    const int x = in / (width * p.splits), rest = in - x * width * p.splits;
    Work w;
    int pair;
    if (finder.find(x, w, pair)) {
      w.kvh = sec * p.section + rest % width;
      w.split = rest / width;
      w.i0 = pair * 2 * p.tq;
      int n[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int first = w.i0 + t * p.tq;
        const int last = min(first + p.tq, w.lq) - 1;  // last live token
        int keys = p.causal ? min(w.lk, last + w.lk - w.lq + 1) : w.lk;
        if (last < first) keys = 0;
        n[t] = keys > 0 ? (keys + kTile - 1) / kTile : 0;
      }
      const int n_max = max(n[0], n[1]);
      w.j0 = 0;
      w.j1 = n_max;
      if (p.splits > 1) {  // at most 32 splits of 2^24 tiles
        w.j0 = w.split * n_max / p.splits;
        w.j1 = (w.split + 1) * n_max / p.splits;
      }
      w.end[0] = min(w.j1, n[0]);
      w.end[1] = min(w.j1, n[1]);
      const uint32_t slot = count & 1u;
      if (!warp_wait(smem_u32(&bars->work_empty[slot]), ((count >> 1) & 1u) ^ 1u, abort_flag,
                     p.status, kDevTimeoutProducer))
        return;  // nothing more is handed out: the others' waits run out
      if (lane < 9) reinterpret_cast<uint32_t *>(&bars->marks[count % 3])[lane] = 0u;
      __syncwarp();
      if (lane == 0) {
        bars->work[slot] = w;
        mbar_arrive(smem_u32(&bars->work_full[slot]));
      }
      __syncwarp();
      ++count;
    }
    if (!warp_wait(smem_u32(&bars->cancel_full), asked & 1u, abort_flag, p.status,
                   kDevTimeoutProducer))
      return;
    idx = cancelled_block(response);
    fence_proxy_async_smem();  // read before the next response is written
    __syncwarp();
  }
  const uint32_t slot = count & 1u;
  if (!warp_wait(smem_u32(&bars->work_empty[slot]), ((count >> 1) & 1u) ^ 1u, abort_flag,
                 p.status, kDevTimeoutProducer))
    return;
  if (lane == 0) {
    bars->work[slot].kvh = -1;
    mbar_arrive(smem_u32(&bars->work_full[slot]));
  }
}

// The k-th unit of this CTA; false when there is none left.  The wait ends
// by its own time limit only: the two warps of a row both get the unit or
// both give up.
__device__ __forceinline__ bool next_work(Bars *bars, uint32_t k, int lane, int *status, Work &w) {
  volatile int no_abort = 0;
  const uint32_t slot = k & 1u;
  if (!warp_wait(smem_u32(&bars->work_full[slot]), (k >> 1) & 1u, &no_abort, status,
                 kDevTimeoutProducer)) {
    *const_cast<volatile int *>(&bars->abort_flag) = 1;
    return false;
  }
  w = bars->work[slot];
  __syncwarp();
  if (lane == 0) mbar_arrive(smem_u32(&bars->work_empty[slot]));
  return w.kvh >= 0;
}

// Value tiles at the edge of what a unit's rows see, between their load (v_raw) and
// the products (v_full).
template <typename T, int kDqk, int kDv>
__device__ __forceinline__ void edge_role(const Params &p, Bars *bars, uint8_t *smem, int lane) {
  using PL = Plan<kDqk, kDv>;
  volatile int *abort_flag = &bars->abort_flag;
  uint32_t tile = 0, raw = 0;  // V tiles so far; bit st: parity of stage st's next v_raw phase
  Work w;
  for (uint32_t k = 0; next_work(bars, k, lane, p.status, w); ++k) {
    if (PL::kRowsClear) continue;
    const Seen seen = seen_keys(p, w);
    for (int j = max(seen.all / kTile, w.j0); j < w.j1; ++j) {
      const uint32_t st = (tile + (j - w.j0)) % PL::kVStages;
      if (!warp_wait(smem_u32(&bars->v_raw[st]), (raw >> st) & 1u, abort_flag, p.status,
                     kDevTimeoutProducer))
        return;
      raw ^= 1u << st;
      const int r0 = max(seen.all - j * kTile, 0), r1 = min(max(seen.some - j * kTile, r0), kTile);
      clear_hidden<T, PL::kVChunks, PL::kChunkBytes, 4>(smem + PL::kOffV + st * PL::kVBytes, r0, r1,
                                                        j * kTile - seen.all, bars->marks[k % 3],
                                                        lane, 32);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars->v_full[st]));
    }
    tile += max(w.j1 - w.j0, 0);
  }
}

template <typename T, int kDqk, int kDv>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap q_map,
                            const __grid_constant__ CUtensorMap k_map,
                            const __grid_constant__ CUtensorMap v_map,
                            const __grid_constant__ Params p) {
  using PL = Plan<kDqk, kDv>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles need it
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, kDevBadSmemAlign);
    return;
  }
  Bars *bars = reinterpret_cast<Bars *>(smem);
  volatile int *abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;

  // the scheduler's first reads, on their way while the CTA sets up
  if (warp == kSchedulerWarp && lane < min(p.batch, 32)) {
    asm volatile("prefetch.global.L1 [%0];" ::"l"(p.cu_q + lane));
    asm volatile("prefetch.global.L1 [%0];" ::"l"(p.cu_k + lane));
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&bars->k_full[i]), 1);
      mbar_init(smem_u32(&bars->k_empty[i]), 2);  // by each Q tile's stream
      mbar_init(smem_u32(&bars->v_full[i]), 1);
      mbar_init(smem_u32(&bars->v_raw[i]), 1);
      mbar_init(smem_u32(&bars->v_empty[i]), 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->q_full[i]), 1);
      mbar_init(smem_u32(&bars->q_empty[i]), 1);
      mbar_init(smem_u32(&bars->s_full[i]), 1);
      mbar_init(smem_u32(&bars->p_full[i][0]), 8);
      mbar_init(smem_u32(&bars->p_full[i][1]), 8);
      mbar_init(smem_u32(&bars->o_full[i]), 1);
      mbar_init(smem_u32(&bars->work_full[i]), 1);
      mbar_init(smem_u32(&bars->work_empty[i]), kRowWarps + 4);  // rows, producer, edge, MMA twice
    }
    mbar_init(smem_u32(&bars->cancel_full), 1);
    mbar_init(smem_u32(&bars->drain), 1);
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&bars->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const uint32_t qbase = smem_u32(smem + PL::kOffQ), kbase = smem_u32(smem + PL::kOffK),
                 vbase = smem_u32(smem + PL::kOffV);

  if (warp < kRowWarps) {
    take_registers<kRowRegs>();
    uint32_t steps = 0, outs = 0, tiles = 0;
    Work it;
    for (uint32_t k = 0; next_work(bars, k, lane, p.status, it); ++k) {
      row_role<T, kDqk, kDv>(p, it, bars, smem, tmem, warp, lane, steps, outs, k, tiles);
      tiles += max(it.j1 - it.j0, 0);
    }
  } else if (warp == kSchedulerWarp) {
    give_registers<kOtherRegs>();
    scheduler_role(p, bars, lane);
  } else if (warp == kEdgeWarp) {
    give_registers<kOtherRegs>();
    edge_role<T, kDqk, kDv>(p, bars, smem, lane);
  } else if (warp == kProducerWarp) {
    give_registers<kOtherRegs>();
    uint32_t g = 0, gv = 0, gq[2] = {0, 0};  // K tiles, V tiles, Q tiles issued
    uint32_t raw = 0, to_raw = 0;  // bit st: v_raw phases of stage st (parity); its last tile's
    if (lane == 0) {
      tma_prefetch_desc(&q_map);
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
    Work it{};
    bool ok = true;
    auto load_q = [&](int x) {
      if (it.end[x] <= it.j0) return;
      if (!(ok = warp_wait(smem_u32(&bars->q_empty[x]), (gq[x] & 1u) ^ 1u, abort_flag, p.status,
                           kDevTimeoutProducer)))
        return;
      if (lane == 0) {
        const uint32_t qf = smem_u32(&bars->q_full[x]);
        mbar_arrive_expect_tx(qf, PL::kQkChunks * p.tq * p.group * 128);
#pragma unroll
        for (int ch = 0; ch < PL::kQkChunks; ++ch)
          tma_load_3d(qbase + x * PL::kQBytes + ch * PL::kChunkBytes, &q_map, qf, ch * 64,
                      it.kvh * p.group, it.q0 + it.i0 + x * p.tq);
      }
      ++gq[x];
    };
    for (uint32_t k = 0; ok && next_work(bars, k, lane, p.status, it); ++k) {
      if (it.j1 <= it.j0) continue;
      // first tile that the edge warp has to look at
      const int edge = PL::kRowsClear ? INT32_MAX : seen_keys(p, it).all / kTile;
      load_q(0);
      for (int j = it.j0; ok && j < it.j1; ++j) {
        const uint32_t ks = g % PL::kKStages, vs = gv % PL::kVStages;
        if (!(ok = warp_wait(smem_u32(&bars->k_empty[ks]), ((g / PL::kKStages) & 1u) ^ 1u,
                             abort_flag, p.status, kDevTimeoutProducer)))
          break;
        if (lane == 0) {
          const uint32_t kf = smem_u32(&bars->k_full[ks]);
          mbar_arrive_expect_tx(kf, PL::kKBytes);
#pragma unroll
          for (int ch = 0; ch < PL::kQkChunks; ++ch)
            tma_load_3d(kbase + ks * PL::kKBytes + ch * PL::kChunkBytes, &k_map, kf, ch * 64,
                        it.k0 + j * kTile, it.kvh);
        }
        ++g;
        if (j == it.j0) {  // Q tile 1 of the last unit may be in use a little longer
          load_q(1);
          if (!ok) break;
        }
        if (!(ok = warp_wait(smem_u32(&bars->v_empty[vs]), ((gv / PL::kVStages) & 1u) ^ 1u,
                             abort_flag, p.status, kDevTimeoutProducer)))
          break;
        to_raw = (to_raw & ~(1u << vs)) | static_cast<uint32_t>(j >= edge) << vs;
        if (j >= edge) raw ^= 1u << vs;
        if (lane == 0) {
          const uint32_t vf = smem_u32(j >= edge ? &bars->v_raw[vs] : &bars->v_full[vs]);
          mbar_arrive_expect_tx(vf, PL::kVBytes);
#pragma unroll
          for (int ch = 0; ch < PL::kVChunks; ++ch)
            tma_load_3d(vbase + vs * PL::kVBytes + ch * PL::kChunkBytes, &v_map, vf, ch * 64,
                        it.k0 + j * kTile, it.kvh);
        }
        ++gv;
      }
    }
    if (*abort_flag) {
      // copies in flight must land before the CTA may exit
      volatile int never = 0;
      for (int x = 0; x < 2; ++x)
        if (gq[x]) wait_inline(smem_u32(&bars->q_full[x]), (gq[x] - 1) & 1u, &never, nullptr, 0);
      for (uint32_t t = g > PL::kKStages ? g - PL::kKStages : 0; t < g; ++t)
        wait_inline(smem_u32(&bars->k_full[t % PL::kKStages]), (t / PL::kKStages) & 1u, &never,
                    nullptr, 0);
      for (uint32_t t = gv > PL::kVStages ? gv - PL::kVStages : 0; t < gv; ++t) {
        const uint32_t st = t % PL::kVStages;
        if (to_raw >> st & 1u)
          wait_inline(smem_u32(&bars->v_raw[st]), (raw >> st & 1u) ^ 1u, &never, nullptr, 0);
        else
          wait_inline(smem_u32(&bars->v_full[st]), (t / PL::kVStages) & 1u, &never, nullptr, 0);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------- MMA issuer
    give_registers<kOtherRegs>();
    constexpr uint32_t kIdescQK = umma_idesc_f16(128, kTile, fmt, 0);
    constexpr uint32_t kIdescPV = umma_idesc_f16(128, kDv, fmt, 1);
    const uint64_t q_desc = smem_desc_swz(qbase, 16, 1024, 2);
    const uint64_t k_desc = smem_desc_swz(kbase, 16, 1024, 2);
    const uint64_t v_desc = smem_desc_swz(vbase, PL::kChunkBytes, 1024, 2);
    auto ready = [&](const uint64_t *bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_probe(smem_u32(bar), parity)) != 0;
    };
    // S of Q tile x and the key tile in stage st
    auto issue_qk = [&](int x, uint32_t st) {
      const uint64_t qd = q_desc + static_cast<uint64_t>((x * PL::kQBytes) >> 4);
      const uint64_t kd = k_desc + static_cast<uint64_t>((st * PL::kKBytes) >> 4);
#pragma unroll
      for (int ch = 0; ch < PL::kQkChunks; ++ch)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint64_t off = static_cast<uint64_t>((ch * PL::kChunkBytes + kk * 32) >> 4);
          umma_ss_warp(tmem + PL::kColS + x * kTile, qd + off, kd + off, kIdescQK,
                       (ch | kk) ? 1u : 0u);
        }
      tc_commit_warp(smem_u32(&bars->s_full[x]));
    };
    // value product with the tile in stage st: K steps (16 keys each) 0 to 2 of
    // both halves (part 0), or the last ones
    auto issue_pv = [&](int x, uint32_t st, int part, bool first) {
      const uint64_t vd = v_desc + static_cast<uint64_t>((st * PL::kVBytes) >> 4);
#pragma unroll
      for (int i = part ? 3 : 0; i < (part ? 4 : 3); ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          umma_ts_warp(tmem + PL::kColO + x * kDv,
                       tmem + PL::kColS + x * kTile + half * (kTile / 2) + i * 8,
                       vd + static_cast<uint64_t>(((half * 4 + i) * 16 * 128) >> 4), kIdescPV,
                       (first && i == 0 && half == 0) ? 0u : 1u);
    };
    // The two Q tiles are independent streams of products, each waiting for
    // its own rows: one tile's next unit starts while the other still ends
    // its last.  While both wait for their rows they are served in turn.
    //
    // A parity wait tells a phase from the one before it only, so a stream sees
    // every K and every V tile land, in order, and releases each itself: those it
    // multiplies when their products are done, those it has no step for
    // as soon as they land (walk).  Where rows look at V tile t themselves, its
    // scores are issued once tile t - 1 has been seen, so that an earlier phase can not
    // answer their wait either.
    enum Need { kUnit, kQK, kP, kNone };
    struct Stream {
      Need need = kUnit;
      uint32_t unit = 0, q = 0, steps = 0;  // units, Q tiles begun; P taken
      uint32_t g = 0, k = 0, v = 0;  // first tile of the unit; next K, V tile to see
      int i = 0, left = 0, n = 0;    // step; steps of this tile, of the unit
    } st0, st1;
    auto k_landed = [&](uint32_t t) {
      return ready(&bars->k_full[t % PL::kKStages], (t / PL::kKStages) & 1u);
    };
    auto v_landed = [&](uint32_t t) {
      return ready(&bars->v_full[t % PL::kVStages], (t / PL::kVStages) & 1u);
    };
    // tiles before the unit's first that the stream has no step for, V after K:
    // none is left when v has come to g
    auto walk = [&](Stream &s) -> bool {
      bool moved = false;
      while (s.k < s.g && k_landed(s.k)) {
        if (lane == 0) mbar_arrive(smem_u32(&bars->k_empty[s.k % PL::kKStages]));
        ++s.k;
        moved = true;
      }
      while (s.v < s.g && s.v < s.k && v_landed(s.v)) {
        if (lane == 0) mbar_arrive(smem_u32(&bars->v_empty[s.v % PL::kVStages]));
        ++s.v;
        moved = true;
      }
      return moved;
    };
    // whatever needs no rows: the next unit, the next scores
    auto feed = [&](int x, Stream &s) -> bool {
      bool moved = false;
      while (s.need == kUnit) {
        const uint32_t slot = s.unit & 1u;
        if (!ready(&bars->work_full[slot], (s.unit >> 1) & 1u)) break;
        const Work &w = bars->work[slot];
        const bool none = w.kvh < 0;
        s.i = 0;
        s.n = none ? 0 : w.j1 - w.j0;
        s.left = none ? 0 : max(w.end[x] - w.j0, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->work_empty[slot]));
        ++s.unit;
        s.need = none ? kNone : (s.left > 0 ? kQK : kUnit);
        if (s.need == kUnit) s.g += s.n;
        moved = true;
      }
      moved |= walk(s);
      if (s.need == kQK) {
        const uint32_t t = s.g + s.i;
        if (s.k < t || (PL::kRowsClear && s.v < t)) return moved;
        if (s.i == 0 && !ready(&bars->q_full[x], s.q & 1u)) return moved;
        if (!k_landed(t)) return moved;
        tc_fence_after();
        issue_qk(x, t % PL::kKStages);
        tc_commit_warp(smem_u32(&bars->k_empty[t % PL::kKStages]));
        ++s.k;
        if (s.i == s.left - 1) {
          tc_commit_warp(smem_u32(&bars->q_empty[x]));
          ++s.q;
        }
        s.need = kP;
        moved = true;
      }
      return moved;
    };
    auto wait = [&](const uint64_t *bar, uint32_t parity) {
      return warp_wait(smem_u32(bar), parity, abort_flag, p.status, kDevTimeoutMma);
    };
    // the first part of this step's P is there (or waited for); then its value
    // product and the next scores
    auto serve = [&](int x, Stream &s) -> bool {
      const uint32_t vs = s.v % PL::kVStages;
      if (!wait(&bars->p_full[x][0], s.steps & 1u)) return false;
      tc_fence_after();
      issue_pv(x, vs, 0, s.i == 0);
      if (!wait(&bars->p_full[x][1], s.steps & 1u)) return false;
      tc_fence_after();
      issue_pv(x, vs, 1, false);
      ++s.steps;
      if (s.i == s.left - 1) tc_commit_warp(smem_u32(&bars->o_full[x]));
      tc_commit_warp(smem_u32(&bars->v_empty[vs]));
      ++s.v;
      s.need = ++s.i < s.left ? kQK : kUnit;
      if (s.need == kUnit) s.g += s.n;
      feed(x, s);
      return true;
    };
    int turn = 0;
    long long idle = 0;  // since when nothing has moved (0: it has)
    while (st0.need != kNone || st1.need != kNone) {
      // A tile can be served once its V tile is there: a tile that is ahead of
      // the other waits for stages the other has yet to release, so the issuer
      // must not block on it.
      auto v_ready = [&](const Stream &s) { return s.v == s.g + s.i && v_landed(s.v); };
      const bool w0 = st0.need == kP && v_ready(st0), w1 = st1.need == kP && v_ready(st1);
      // serve tile 0 / 1 (blocking on its rows): its turn while both could be,
      // or the other has no work left; otherwise only when its rows are done
      const bool go0 = w0 && (w1 ? turn == 0 : st1.need == kNone ||
                                                   ready(&bars->p_full[0][0], st0.steps & 1u));
      const bool go1 = !go0 && w1 && (w0 ? turn == 1 : st0.need == kNone ||
                                                           ready(&bars->p_full[1][0], st1.steps & 1u));
      if (go0) {
        if (!serve(0, st0)) break;
        turn = 1;
      } else if (go1) {
        if (!serve(1, st1)) break;
        turn = 0;
      }
      bool moved = go0 || go1;
      // only what each can do now: the loop's length is in every step's chain
      if (st0.need < kP) moved |= feed(0, st0);
      else if (st0.v < st0.g) moved |= walk(st0);
      if (st1.need < kP) moved |= feed(1, st1);
      else if (st1.v < st1.g) moved |= walk(st1);
      if (moved) {
        idle = 0;
        continue;
      }
      const long long now = clock64();
      if (idle == 0) idle = now;
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
      if (__any_sync(0xffffffffu, now - idle > kWaitLimitCycles)) {
        *abort_flag = 1;
        if (lane == 0 && p.status) atomicExch(p.status, kDevTimeoutMma);
        break;
      }
    }
    __syncwarp();
    // every issued MMA must finish before TMEM is released
    tc_commit_warp(smem_u32(&bars->drain));
    volatile int never = 0;
    wait_inline(smem_u32(&bars->drain), 0, &never, p.status, kDevTimeoutDrain);
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Merge of a row's partial results (splits > 1), one warp per row.
template <typename T>
__global__ void __launch_bounds__(128) prompt_merge_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int64_t rows = static_cast<int64_t>(p.hq) * p.total_q;
  if (row >= rows) return;
  const int head = static_cast<int>(row / p.total_q), tok = static_cast<int>(row % p.total_q);
  if (tok >= __ldg(p.cu_q + p.batch)) return;  // of no sequence: not written
  const int lane = threadIdx.x & 31;
  RowSum<1> st;
  st.init();
  st.fold<4>(p.part_o, p.part_lse, 0, 1, p.splits, p.d_v, lane,
             [&](int s) { return static_cast<int64_t>(s) * rows + row; });
  const float l = st.finish(
      static_cast<T *>(p.o) + static_cast<int64_t>(tok) * p.o_st + head * p.o_sh, p.d_v, lane);
  if (p.lse && lane == 0) p.lse[row] = l;
}

template <typename T, int kDqk, int kDv>
cudaError_t launch_t(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm,
                     const Params &p, unsigned grid, cudaStream_t stream) {
  auto kern = prompt_attention_kernel<T, kDqk, kDv>;
  constexpr int smem = Plan<kDqk, kDv>::kSmemBytes;
  // registers that the row warps take must have been given up by the others
  static const bool fits = [&] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess &&
           a.numRegs * kThreads >= 32 * (kRowWarps * kRowRegs + (kThreads / 32 - kRowWarps) * kOtherRegs);
  }();
  if (!fits) return cudaErrorInvalidConfiguration;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, smem, stream>>>(qm, km, vm, p);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.hq) * p.total_q + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, prompt_merge_kernel<T>, p);
}

template <typename T>
cudaError_t launch_d(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm,
                     const Params &p, int d_qk, unsigned grid, cudaStream_t stream) {
  if (d_qk > 128) return launch_t<T, 192, 128>(qm, km, vm, p, grid, stream);
  if (d_qk > 64 || p.d_v > 64) return launch_t<T, 128, 128>(qm, km, vm, p, grid, stream);
  return launch_t<T, 64, 64>(qm, km, vm, p, grid, stream);
}

}  // namespace prompt

// Tokens of one Q tile: as many as fit 128 rows with the group's heads.
int prompt_tile_tokens(const fa_prompt_args *a) {
  return prompt::kTile / (a->num_q_heads / a->num_kv_heads);
}

// Upper bound of the (sequence, Q tile pair) items: the sum over sequences of
// ceil(tokens / span) with span = the tokens of a pair.
int64_t prompt_items(const fa_prompt_args *a) {
  return a->total_q / (2 * prompt_tile_tokens(a)) + a->batch;
}

// Units an item's keys are cut into when there are fewer items than SMs (few
// new tokens over many keys).  In steps of one key tile (about 1.7 us): a unit
// of n tiles costs n + 4, units run in rounds of one per SM, and the partial
// rows are written and read once.  The count with the lowest estimate.
int prompt_splits(const fa_prompt_args *a, int sms) {
  const int64_t span = 2 * prompt_tile_tokens(a);
  const int64_t items = std::max<int64_t>((a->total_q + span - 1) / span, a->batch);
  const int64_t units = items * a->num_kv_heads;
  if (units >= sms || a->batch == 0) return 1;
  const int64_t seen = a->causal ? a->total_k - std::min(a->total_q, a->total_k) / 2 : a->total_k;
  const int64_t tiles = seen / a->batch / prompt::kTile;
  const double row_bytes = 8.0 * a->num_q_heads * a->total_q * a->d_v;  // written and read, f32
  int best = 1;
  double best_cost = static_cast<double>(tiles + 4);
  for (int s = 2; s <= 32 && tiles / s >= 4; ++s) {
    const double rounds = static_cast<double>((units * s + sms - 1) / sms);
    const double cost =
        rounds * (static_cast<double>(tiles) / s + 4) + 2 + s * row_bytes / (1.7 * 5.0e6);
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

cudaError_t launch_prompt(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm,
                          const fa_prompt_args *a, int splits, float *part_o, float *part_lse,
                          cudaStream_t stream) {
  prompt::Params p;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  p.batch = a->batch;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
  p.v = a->v;
  p.v_st = a->v_stride_t;
  p.v_sh = a->v_stride_h;
  p.hq = a->num_q_heads;
  p.hkv = a->num_kv_heads;
  p.group = a->num_q_heads / a->num_kv_heads;
  p.tq = prompt_tile_tokens(a);
  p.d_v = a->d_v;
  p.causal = a->causal;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.o = a->o;
  p.o_st = a->o_stride_t;
  p.o_sh = a->o_stride_h;
  p.lse = a->lse;
  p.status = a->status;
  p.items = static_cast<int32_t>(prompt_items(a));
  p.splits = splits;
  p.part_o = part_o;
  p.part_lse = part_lse;
  // kv heads at a time whose keys and values stay in L2 (half of 126 MB)
  const int64_t head_bytes = static_cast<int64_t>(a->total_k) * (a->d_qk + a->d_v) * 2 + 1;
  p.section = static_cast<int32_t>(
      std::min<int64_t>(std::max<int64_t>((int64_t{63} << 20) / head_bytes, 1), a->num_kv_heads));
  const int64_t grid = static_cast<int64_t>(p.items) * splits * a->num_kv_heads;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return a->dtype == FA_DTYPE_F16
             ? prompt::launch_d<__half>(qm, km, vm, p, a->d_qk, static_cast<unsigned>(grid), stream)
             : prompt::launch_d<__nv_bfloat16>(qm, km, vm, p, a->d_qk,
                                               static_cast<unsigned>(grid), stream);
}

}  // namespace fa
