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
// causal diagonal wastes few columns.  Both Q tiles walk the item's key tiles
// of 128 together, in opposite phase: while the tensor pipe computes one
// tile's products, the other tile's warps take the exponentials.  Per tile
// and step the tensor pipe needs 2 * 128 * 128 * (d_qk + d_v) flops at 8192 a
// cycle (1024 cycles at head size 128) and the exponentials 128 * 128 at 16 a
// cycle (1024 cycles), so neither may wait for the other.
//
//   warps 0-7 / 8-15: rows of Q tile 0 / 1 (two threads per row, S read from
//     TMEM, P written over it as the A operand of P V)
//   warp 16: MMA issuer    warp 17: TMA producer
//
// TMEM: S0 S1 (128 columns each, P in place), O0 O1.  The issuer's stream is
// in order, so the barrier that announces S of step j also says that P V of
// step j - 1 is complete: the rows rescale O without a further wait.
//
// Every mbarrier wait is bounded (common.cuh).
#include "common.cuh"
#include "flagattn_b200.h"

namespace fa {
namespace prompt {

// Two warps beyond the roles fill up the last warpgroup, which gives its
// registers to the row warps: 16 * 112 + 4 * 32 = 20 * 96, the launch's.
constexpr int kThreads = 640, kRowRegs = 112, kOtherRegs = 32;
constexpr int kRowWarps = 16, kMmaWarp = 16, kProducerWarp = 17;
// Of every 8 pairs of columns this many take their exponentials on the FMA
// pipes instead of the special-function unit.
constexpr int kFmaPairs = 2;
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
  static constexpr int kOffX = 1024;
  static constexpr int kOffQ = 3072;
  static constexpr int kOffK = kOffQ + 2 * kQBytes;
  static constexpr int kOffV = kOffK + kKStages * kKBytes;
  static constexpr int kSmemUsed = kOffV + kVStages * kVBytes;
  static constexpr int kSmemBytes = kSmemUsed;
  static constexpr uint32_t kColS = 0, kColO = 2 * kTile;
  static_assert(kColO + 2 * kDv <= kTmemCols, "TMEM plan");
  static_assert(kSmemBytes <= 232448, "shared memory plan exceeds 227 KB");
};

struct Bars {
  uint64_t q_full;
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2], o_full[2];
  uint64_t p_full[2][2];  // [Q tile][first / last 32 columns of both halves]
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  int warp_sum[kThreads / 32];
  int item_seq, item_tile;  // -1: no work
};
// Row maxima, at the end row sums, that the two threads of a row exchange.
struct Exchange {
  float v[2][2][kTile];  // [Q tile][half][row]
};
static_assert(sizeof(Exchange) == 2048, "exchange block");
static_assert(sizeof(Bars) <= 1024, "barrier block");

struct Params {
  const int32_t *cu_q, *cu_k;
  int32_t batch, total_q, total_k, hq, hkv, group, tq;  // tq: tokens of a Q tile
  int32_t d_v, causal;
  float scale_log2;
  void *o;
  int64_t o_st, o_sh;
  float *lse;  // nullable, [hq][total_q]
  int *status;
};

// Rows [start, end) of sequence b in a packed tensor of `total` rows; offsets
// outside it or out of order are cut to what exists.
__device__ __forceinline__ void seq_range(const int32_t *cu, int b, int total, int &start,
                                          int &len) {
  start = min(max(__ldg(cu + b), 0), total);
  len = min(max(__ldg(cu + b + 1), start), total) - start;
}

// Sequence and Q-tile pair of item x: sequences in order, each from its last
// pair (under a causal mask the one with most keys) to its first.  All
// threads take part.
__device__ __forceinline__ void find_item(const Params &p, int x, Bars *bars) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  const int span = 2 * p.tq;
  int local = 0;
  for (int b = b0; b < b1; ++b) {
    int s, n;
    seq_range(p.cu_q, b, p.total_q, s, n);
    local += (n + span - 1) / span;
  }
  int incl = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) bars->warp_sum[warp] = incl;
  __syncthreads();
  int run = incl - local;
  for (int w = 0; w < warp; ++w) run += bars->warp_sum[w];
  if (x >= run && x < run + local) {
    for (int b = b0; b < b1; ++b) {
      int s, n;
      seq_range(p.cu_q, b, p.total_q, s, n);
      const int tiles = (n + span - 1) / span;
      if (x < run + tiles) {
        bars->item_seq = b;
        bars->item_tile = tiles - 1 - (x - run);
        break;
      }
      run += tiles;
    }
  }
  __syncthreads();
}

struct Item {
  int kvh, q0, lq, k0, lk, i0;  // i0: first token of Q tile 0 in its sequence
  int n[2];                     // key tiles of each Q tile
};

__device__ __forceinline__ Item get_item(const Params &p, int kvh, int b, int pair) {
  Item it;
  it.kvh = kvh;
  seq_range(p.cu_q, b, p.total_q, it.q0, it.lq);
  seq_range(p.cu_k, b, p.total_k, it.k0, it.lk);
  it.i0 = pair * 2 * p.tq;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int first = it.i0 + x * p.tq;
    const int last = min(first + p.tq, it.lq) - 1;  // last live token
    int keys = p.causal ? min(it.lk, last + it.lk - it.lq + 1) : it.lk;
    if (last < first) keys = 0;
    it.n[x] = keys > 0 ? (keys + kTile - 1) / kTile : 0;
  }
  return it;
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

// 2^x for kN pairs of x >= -126 without the special-function unit: x = n + f
// with n the nearest integer (adding 1.5 * 2^23 leaves n in the low mantissa
// bits), 2^f by a polynomial of degree 4 (minimax in relative error on [-1/2,
// 1/2], Remez exchange: 2.6e-6, below the rounding of P to 16 bits), n added
// to the exponent field.  Written step by step over all pairs: the chains are
// independent and hide one another's latency.
template <int kN>
__device__ __forceinline__ void exp2_pairs(uint64_t (&x)[kN]) {
  constexpr float kMagic = 12582912.f;
  const float k[5] = {0.9999992847442627f, 0.6931217908859253f, 0.240247443318367f,
                      0.05591785907745361f, 0.009570102207362652f};
  const uint64_t magic = f32x2(kMagic, kMagic);
  uint64_t r[kN], y[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) r[i] = fadd2(x[i], magic);
#pragma unroll
  for (int i = 0; i < kN; ++i) y[i] = fadd2(r[i], f32x2(-kMagic, -kMagic));
#pragma unroll
  for (int i = 0; i < kN; ++i) x[i] = ffma2(y[i], f32x2(-1.f, -1.f), x[i]);
#pragma unroll
  for (int i = 0; i < kN; ++i) y[i] = ffma2(x[i], f32x2(k[4], k[4]), f32x2(k[3], k[3]));
#pragma unroll
  for (int d = 2; d >= 0; --d)
#pragma unroll
    for (int i = 0; i < kN; ++i) y[i] = ffma2(y[i], x[i], f32x2(k[d], k[d]));
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float r0, r1, y0, y1;
    f32x2_split(r[i], r0, r1);
    f32x2_split(y[i], y0, y1);
    x[i] = f32x2(__uint_as_float(__float_as_uint(y0) + (__float_as_uint(r0) << 23)),
                 __uint_as_float(__float_as_uint(y1) + (__float_as_uint(r1) << 23)));
  }
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

// Rows of Q tile x: two threads per row, each with half of the key tile's
// columns (`half`) and of O's.  A wait that gives up does not end the loop
// (every wait returns at once from then on): the two warps of a row keep
// meeting at their named barrier.
template <typename T, int kDqk, int kDv>
__device__ __forceinline__ void row_role(const Params &p, const Item &it, Bars *bars,
                                         uint8_t *smem, uint32_t tmem, int warp, int lane) {
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
  const int n = it.n[x];
  float m_use = -INFINITY, l = 0.f;
  const uint64_t c2 = f32x2(p.scale_log2, p.scale_log2);
  for (int j = 0; j < n; ++j) {
    warp_wait(smem_u32(&bars->s_full[x]), j & 1u, abort_flag, p.status, kDevTimeoutSoftmax);
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
    bool resc = false;
    float alpha = 1.f;
    if (barrier_any(meet, 64, j == 0 || m_row * p.scale_log2 > m_use + kRescaleThreshold)) {
      *mine = m_row;
      named_bar_sync(meet, 64);
      m_row = max3_nan(m_row, *other, *other);
      named_bar_sync(meet, 64);  // read before the next exchange writes
      const float m_tile = m_row * p.scale_log2;
      if (j == 0) {
        m_use = m_tile;
      } else if (m_tile > m_use + kRescaleThreshold) {
        resc = m_use != -INFINITY;  // O is all zeros while no key was visible
        alpha = resc ? fast_exp2(m_use - m_tile) : 0.f;
        l *= alpha;
        m_use = m_tile;
      }
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
    // Value rows past the sequence's end belong to the next sequence and may
    // hold infinities or NaN; P is 0 there but 0 * NaN is not: clear them.
    // The first Q tile that uses this V tile does so (its P V goes first).
    if (quad == 0 && half == 0 && it.lk < (j + 1) * kTile && (x == 0 || j >= it.n[0])) {
      const int st = j % PL::kVStages;
      warp_wait(smem_u32(&bars->v_full[st]), (j / PL::kVStages) & 1u, abort_flag, p.status,
                kDevTimeoutSoftmax);
      const uint32_t tile = smem_u32(smem + PL::kOffV) + st * PL::kVBytes;
      const int r0 = it.lk - j * kTile;
      const int units = (kTile - r0) * 8;  // 16-byte units of a chunk's rows
      for (int u = lane; u < units * PL::kVChunks; u += 32)
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                         tile + (u / units) * PL::kChunkBytes + r0 * 128 + (u % units) * 16),
                     "r"(0u)
                     : "memory");
      fence_proxy_async_smem();
    }
    const float msafe = m_use == -INFINITY ? 0.f : m_use;
    const uint64_t nm2 = f32x2(-msafe, -msafe);
    uint64_t acc2 = f32x2(0.f, 0.f), acc2b = f32x2(0.f, 0.f);
    // P over S in place, 32 columns at a time
    // kPairs pairs of columns of v from the first on, to words of w
    auto exps = [&](auto fma_pairs, const float *v, uint32_t *w) {
      constexpr int kF = decltype(fma_pairs)::value;  // the first pairs go to the FMA pipes
      constexpr int kPairs = 8;
      uint64_t y[kPairs];
#pragma unroll
      for (int c = 0; c < kPairs; ++c) y[c] = ffma2(f32x2(v[2 * c], v[2 * c + 1]), c2, nm2);
#pragma unroll
      for (int c = kF; c < kPairs; ++c) {
        float x0, x1;
        f32x2_split(y[c], x0, x1);
        y[c] = f32x2(fast_exp2(x0), fast_exp2(x1));
      }
      if constexpr (kF > 0) {
        uint64_t z[kF];
#pragma unroll
        for (int c = 0; c < kF; ++c) {
          float x0, x1;
          f32x2_split(y[c], x0, x1);
          z[c] = f32x2(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
        }
        exp2_pairs<kF>(z);
#pragma unroll
        for (int c = 0; c < kF; ++c) y[c] = z[c];
      }
#pragma unroll
      for (int c = 0; c < kPairs; ++c) {
        float p0, p1;
        f32x2_split(y[c], p0, p1);
        w[c] = Elem<T>::pack2(p0, p1);
        if (c & 1)
          acc2b = fadd2(acc2b, y[c]);
        else
          acc2 = fadd2(acc2, y[c]);
      }
    };
    // P of 32 columns (and the rescaled O, the cleared V) is there: the value
    // product of the first columns starts while the last are computed
    auto hand_over = [&](int part) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars->p_full[x][part]));
    };
    auto all = [&](auto fma_pairs) {
      uint32_t w[16], w2[16];
      exps(fma_pairs, s, w);
      exps(fma_pairs, s + 16, w + 8);
      tmem_st16p(t_s, w);
      exps(fma_pairs, s2, w2);  // hides the store's latency
      hand_over(0);
      exps(fma_pairs, s2 + 16, w2 + 8);
      tmem_st16p(t_s + 16, w2);
      hand_over(1);
    };
    if (masked)  // a masked weight has to be exactly 0
      all(std::integral_constant<int, 0>());
    else
      all(std::integral_constant<int, kFmaPairs>());
    float a0, a1;
    f32x2_split(fadd2(acc2, acc2b), a0, a1);
    l += a0 + a1;
  }
  if (n > 0) {
    *mine = l;
    named_bar_sync(meet, 64);
    l += *other;
    if (!warp_wait(smem_u32(&bars->o_full[x]), 0, abort_flag, p.status, kDevTimeoutSoftmax)) return;
    tc_fence_after();
  }
  const float f = l == 0.f ? 0.f : 1.f / l;  // a NaN stays one
  T *orow = static_cast<T *>(p.o) + static_cast<int64_t>(it.q0 + tok) * p.o_st + head * p.o_sh +
            half * kOCols;
#pragma unroll 1
  for (int c = 0; c < kOCols / 16; ++c) {
    float v[16];
    if (n > 0) {
      tmem_ld16(t_o + 16 * c, v);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (half * kOCols + 16 * c + 8 * i < p.d_v) {
          uint4 u;
          u.x = Elem<T>::pack2(v[8 * i] * f, v[8 * i + 1] * f);
          u.y = Elem<T>::pack2(v[8 * i + 2] * f, v[8 * i + 3] * f);
          u.z = Elem<T>::pack2(v[8 * i + 4] * f, v[8 * i + 5] * f);
          u.w = Elem<T>::pack2(v[8 * i + 6] * f, v[8 * i + 7] * f);
          *reinterpret_cast<uint4 *>(orow + 16 * c + 8 * i) = u;
        }
      }
    }
  }
  if (half == 0 && live && p.lse)
    p.lse[static_cast<int64_t>(head) * p.total_q + it.q0 + tok] =
        l == 0.f ? -INFINITY : (m_use + __log2f(l)) * 0.6931471805599453f;
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

  if (threadIdx.x == 0) bars->item_seq = -1;
  __syncthreads();
  find_item(p, blockIdx.x / p.hkv, bars);
  if (bars->item_seq < 0) return;  // the grid is an upper bound of the items
  const Item it = get_item(p, blockIdx.x % p.hkv, bars->item_seq, bars->item_tile);
  const int n_max = max(it.n[0], it.n[1]);

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bars->q_full), 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&bars->k_full[i]), 1);
      mbar_init(smem_u32(&bars->k_empty[i]), 1);
      mbar_init(smem_u32(&bars->v_full[i]), 1);
      mbar_init(smem_u32(&bars->v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->s_full[i]), 1);
      mbar_init(smem_u32(&bars->p_full[i][0]), 8);
      mbar_init(smem_u32(&bars->p_full[i][1]), 8);
      mbar_init(smem_u32(&bars->o_full[i]), 1);
    }
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
    row_role<T, kDqk, kDv>(p, it, bars, smem, tmem, warp, lane);
  } else if (warp > kProducerWarp) {
    give_registers<kOtherRegs>();
  } else if (warp == kProducerWarp) {
    give_registers<kOtherRegs>();
    int gk = 0, gv = 0, gq = 0;
    if (lane == 0 && n_max > 0) {
      tma_prefetch_desc(&q_map);
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
      const uint32_t qf = smem_u32(&bars->q_full);
      const int qtiles = it.n[1] > 0 ? 2 : 1;
      mbar_arrive_expect_tx(qf, qtiles * PL::kQkChunks * p.tq * p.group * 128);
      gq = 1;
      for (int x = 0; x < qtiles; ++x)
        for (int ch = 0; ch < PL::kQkChunks; ++ch)
          tma_load_3d(qbase + x * PL::kQBytes + ch * PL::kChunkBytes, &q_map, qf, ch * 64,
                      it.kvh * p.group, it.q0 + it.i0 + x * p.tq);
      for (int j = 0; j < n_max; ++j) {
        const int ks = j % PL::kKStages, vs = j % PL::kVStages;
        if (!wait_inline(smem_u32(&bars->k_empty[ks]), ((j / PL::kKStages) & 1u) ^ 1u, abort_flag,
                       p.status, kDevTimeoutProducer))
          break;
        const uint32_t kf = smem_u32(&bars->k_full[ks]);
        mbar_arrive_expect_tx(kf, PL::kKBytes);
        for (int ch = 0; ch < PL::kQkChunks; ++ch)
          tma_load_3d(kbase + ks * PL::kKBytes + ch * PL::kChunkBytes, &k_map, kf, ch * 64,
                      it.k0 + j * kTile, it.kvh);
        ++gk;
        if (!wait_inline(smem_u32(&bars->v_empty[vs]), ((j / PL::kVStages) & 1u) ^ 1u, abort_flag,
                       p.status, kDevTimeoutProducer))
          break;
        const uint32_t vf = smem_u32(&bars->v_full[vs]);
        mbar_arrive_expect_tx(vf, PL::kVBytes);
        for (int ch = 0; ch < PL::kVChunks; ++ch)
          tma_load_3d(vbase + vs * PL::kVBytes + ch * PL::kChunkBytes, &v_map, vf, ch * 64,
                      it.k0 + j * kTile, it.kvh);
        ++gv;
      }
      if (*abort_flag) {
        // copies in flight must land before the CTA may exit
        volatile int never = 0;
        if (gq) wait_inline(qf, 0, &never, nullptr, 0);
        for (int t = max(0, gk - PL::kKStages); t < gk; ++t)
          wait_inline(smem_u32(&bars->k_full[t % PL::kKStages]), (t / PL::kKStages) & 1u, &never,
                    nullptr, 0);
        for (int t = max(0, gv - PL::kVStages); t < gv; ++t)
          wait_inline(smem_u32(&bars->v_full[t % PL::kVStages]), (t / PL::kVStages) & 1u, &never,
                    nullptr, 0);
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
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      return warp_wait(smem_u32(bar), parity, abort_flag, p.status, kDevTimeoutMma);
    };
    // S of Q tile x and key tile j
    auto issue_qk = [&](int x, int j) {
      const uint64_t qd = q_desc + static_cast<uint64_t>((x * PL::kQBytes) >> 4);
      const uint64_t kd = k_desc + static_cast<uint64_t>(((j % PL::kKStages) * PL::kKBytes) >> 4);
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
    // value product of key tile j, K steps of the first (part 0) or last 32
    // columns of each half
    auto issue_pv = [&](int x, int j, int part) {
      const uint64_t vd = v_desc + static_cast<uint64_t>(((j % PL::kVStages) * PL::kVBytes) >> 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kk = (i / 2) * 4 + part * 2 + i % 2;  // 16 keys each
        umma_ts_warp(tmem + PL::kColO + x * kDv,
                     tmem + PL::kColS + x * kTile + (kk / 4) * (kTile / 2) + (kk % 4) * 8,
                     vd + static_cast<uint64_t>((kk * 16 * 128) >> 4), kIdescPV,
                     (j | part | i) ? 1u : 0u);
      }
      if (part == 1 && j == it.n[x] - 1) tc_commit_warp(smem_u32(&bars->o_full[x]));
    };
    if (n_max > 0) ok = wait(&bars->q_full, 0);
    // step j: scores of key tile j, after the value product of tile j - 1
    for (int j = 0; j <= n_max && ok; ++j) {
      if (j < n_max) {
        if (!(ok = wait(&bars->k_full[j % PL::kKStages], (j / PL::kKStages) & 1u))) break;
      }
      if (j > 0) {
        if (!(ok = wait(&bars->v_full[(j - 1) % PL::kVStages], ((j - 1) / PL::kVStages) & 1u)))
          break;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (j > 0 && j - 1 < it.n[x]) {
          if (!(ok = wait(&bars->p_full[x][0], (j - 1) & 1u))) break;
          tc_fence_after();
          issue_pv(x, j - 1, 0);
          if (!(ok = wait(&bars->p_full[x][1], (j - 1) & 1u))) break;
          tc_fence_after();
          issue_pv(x, j - 1, 1);
        }
        if (j < it.n[x]) {
          tc_fence_after();
          issue_qk(x, j);
        }
      }
      if (!ok) break;
      if (j > 0) tc_commit_warp(smem_u32(&bars->v_empty[(j - 1) % PL::kVStages]));
      if (j < n_max) tc_commit_warp(smem_u32(&bars->k_empty[j % PL::kKStages]));
    }
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

template <typename T, int kDqk, int kDv>
cudaError_t launch_t(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm,
                     const Params &p, unsigned grid, cudaStream_t stream) {
  auto kern = prompt_attention_kernel<T, kDqk, kDv>;
  constexpr int smem = Plan<kDqk, kDv>::kSmemBytes;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, smem, stream>>>(qm, km, vm, p);
  return cudaGetLastError();
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

cudaError_t launch_prompt(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm,
                          const fa_prompt_args *a, cudaStream_t stream) {
  prompt::Params p;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  p.batch = a->batch;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
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
  // sum over sequences of ceil(tokens / span) is at most this
  const int64_t items = a->total_q / (2 * p.tq) + a->batch;
  const int64_t grid = items * a->num_kv_heads;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return a->dtype == FA_DTYPE_F16
             ? prompt::launch_d<__half>(qm, km, vm, p, a->d_qk, static_cast<unsigned>(grid), stream)
             : prompt::launch_d<__nv_bfloat16>(qm, km, vm, p, a->d_qk,
                                               static_cast<unsigned>(grid), stream);
}

}  // namespace fa
