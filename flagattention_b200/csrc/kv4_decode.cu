// kv4_decode.cu -- one-token attention over the paged 4-bit cache (kv4.cuh).
//
// For sequence b, query head h of kv head g's group, over the cached tokens t
// with codes c, group minima lo and scales s (G dims each, group index i):
//   q . k_t = sum_i  ks_ti * (sum_{d in i} kc_td q_d) + klo_ti * (sum_{d in i} q_d)
//   o_d     = sum_t (p_t vs_ti) vc_td  +  sum_t p_t vlo_ti
// so codes go to the tensor cores as whole numbers, scales stay f32 factors
// of small tiles, and nothing is expanded to 16-bit rows in memory.
//
// Byte-bound: a token and kv head is D + 8 D / G bytes (144 at D = 128, G =
// 64; 512 in 16 bits).  At the measured copy rate an SM takes about 23 bytes a
// cycle, one 16-token tile of 2304 bytes per 100 cycles, in which its four
// schedulers issue 400 warp instructions and its integer pipes 200: the
// instruction count per tile is the second bound.  mma.sync m16n8k16 (f16)
// fits that: tokens (S = K Q^T) or dims (O^T = V^T P) are the 16 rows, up to 8
// heads the columns, codes come straight from 16-byte loads of global memory into
// A fragments, and P moves between the two products in registers (movmatrix).
// tcgen05 would need the expanded operand written to shared memory first, 4x
// the bytes of the codes.
//
// A code becomes an operand with one AND and no conversion: four bits at the
// bottom of a 16-bit half are the f16 subnormal c * 2^-24, the next four are
// 16 c * 2^-24, both exact in the product; the word's upper codes need one
// shift for four.  2^24 and the factor 16 of every other dim are powers of two
// folded into Q and into the output.  Against two instructions a pair for
// the normal numbers 16 + c (shift, AND-OR) and bf16 operands this took 8
// contexts of up to 65536 tokens from 147 us to 107.
//
// The tensor cores line products up by their operands' exponents, and that of a
// subnormal is 2^-14 however small it is: bits more than 24 below drop out.  A
// product of a lowest code and a query dim 2^k below the largest keeps 15 - k bits
// so, all of a bf16 query's 8 bits up to k = 7 but an f16 query's 11 up to 4 only: scores of
// f16 caches were 2^-21 off.  There every key code goes to bits 4 to 7 (three shifts
// a word, where the time does not change; with bf16, 2^-23 off, they would cost
// 4% of long contexts).
//
// f16 operands hold Q and P' = p * s exactly enough because both are brought
// into its range by a power of two: Q by its row's largest magnitude (bf16 and
// f16 queries then lose nothing above 2^-23 of it), P' by the largest product
// that a warp has met for the head and group of dims.  Small ones are then off by
// 2^-28 of that at most, so neither a large token that has no weight, nor one that only
// another head attends to, nor another group of large values costs accuracy (one
// unit for all heads and groups, by the largest scale: 9% off beside a
// token 10^5 times larger that has no weight).
//
// Four warps of a CTA share a piece (a run of 64-token blocks of one entry),
// one 16-token tile each per block, loaded straight into registers one tile
// ahead while L2 fetches further ones; nothing in the loop meets another warp.
// The pieces are equal shares of all entries' blocks, cut from the sequence
// lengths by every CTA; split entries are merged by a second kernel launched as
// a programmatic dependent.
//
// Scores, sums and the merge are f32.  The tensor cores drop bits of their own
// f32 accumulators, so value sums leave them every 64 tiles.
//
// Measured as graphs of two calls, 64 query / 8 kv heads of 128, groups of 64, bf16: 8
// contexts of 20001 to 65536 tokens 89 us (390 MB read from HBM, 4.4 TB/s; 96 as
// calls), 32 of 1000 to 4096 tokens 30.8 us from L2 and 33.8 with a cold one, one of 700
// tokens 9.3 us (of 8000: 18.3 cold); 64 of 1 to 4001 tokens, 64 / 4 heads of 64, f16: 34.9
// us.  No pipe is full at the long ones (schedulers issue in 56% of the cycles, the
// integer pipe is 55% busy, 64% of the copy rate): 16 warps an SM, each on one
// tile's chain from codes to scores to weights to values, leave gaps.
#include "kv4.cuh"
#include "flagattn_b200.h"
#include "merge.cuh"

namespace fa {
int record_error(int status, const char *msg);

namespace kv4 {
int validate_cache(const fa_kv4_cache *c);
Pool pool_of(const fa_kv4_cache *c);

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kBlockTokens = kWarps * kTileTokens;  // schedule unit: one tile per warp
// P' = p * s * unit, the unit a power of two for each head and group: the largest
// p * s met lands in [2^3, 2^4), and maxima and units move when p passes 2^7 or
// a scale times its unit 2^8, so P' stays below 2^15.
constexpr float kRescaleThreshold = 7.f;
constexpr int kUnitTop = 3, kLimitTop = 8, kUnitMost = 100;
// Stands for "no key yet" as a running maximum: below every finite score, and
// finite, so that differences with it need no special case.
constexpr float kNoMax = -3.0e38f;

struct Params {
  const void *q;
  int64_t q_sb, q_sh;
  Pool pool;
  int32_t num_blocks;
  const int32_t *block_table;
  int64_t bt_stride;
  int32_t bt_width;
  const int32_t *seq_lens;
  int32_t batch, hq, hkv, group;
  int32_t head_tiles;  // entries per kv head: runs of 8 * kNT query heads
  float scale_log2;
  void *o;
  int64_t o_sb, o_sh;
  float *lse;       // nullable [batch][hq]
  float *part_o;    // [slot][8 * kNT][kD]
  float *part_lse;  // [slot][8 * kNT]
  int4 *merge;      // per entry: {first slot or -1, first later slot, later slots, 0}
};

template <int kD, int kGroups, int kNT>
struct Plan {
  static constexpr int kTileB = tile_bytes(kD, kGroups);
  static constexpr int kHeads = 8 * kNT;
  static constexpr int kORow = kD + 4;  // f32 row pitch of the merge buffer (bank spread)
  static constexpr int kMergeBytes = kWarps * kHeads * kORow * 4;
  static_assert(kMergeBytes <= 48 * 1024, "merge buffer");
};
// CTAs per SM: as many as the registers hold without spills in the loop (64
// short chats, head size 64, two head tiles: 34.6 us with four, 32.9 with three;
// 8 long contexts, head size 128, one head tile: 88 us with four, 98 with three).
__host__ __device__ constexpr int blocks_per_sm(int d, int nt) {
  return nt == 1 && d <= 128 ? 4 : (d == 64 ? 3 : 2);
}
// Tiles a warp asks L2 to fetch ahead of the one it loads: 16 warps x 3 x 2304
// bytes in flight cover the latency of HBM (44 KB per SM) several times over.
constexpr int kAhead = 3;

// Units [a0, a1) of the CTA; the first belongs to entry `entry` of sequence b
// (kv heads x head tiles), whose own first unit is x.  CTA p of `parts` starts
// at unit p * chunk + min(p, extra).
struct Share {
  long long a0, a1, x, chunk;
  int b, entry, parts, extra;
};

struct Control {
  long long warp_sum[kWarps];
  Share share;
  float m[kWarps][16], l[kWarps][16];
};

__device__ __forceinline__ int seq_len_of(const Params &p, int b) {
  const int cap = static_cast<int>(
      min(static_cast<long long>(p.bt_width) * p.pool.block_size, 0x7fffff00ll));
  return min(max(__ldg(p.seq_lens + b), 0), cap);
}
__device__ __forceinline__ int blocks_of(int len) { return (len + kBlockTokens - 1) / kBlockTokens; }

// Cost of an entry in units of one block: the blocks, and the start and end of
// a piece (table, first tiles, Q, the warps' merge: about 3 us, three blocks).
constexpr int kPieceCost = 3;

// a / b where the quotient or both numbers are small; the 64-bit division is
// an order of magnitude slower.
__device__ __forceinline__ long long divide(long long a, int b) {
  return a < (1ll << 31) ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// The CTA's share of the work: the entries' costs in entry order, cut into
// `parts` runs that differ by at most one unit.  A thread adds up its run of
// sequences; the one that holds unit a0 finds the entry.
__device__ __forceinline__ void compute_share(const Params &p, Control *ctl) {
  const int B = p.batch, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per_seq = p.hkv * p.head_tiles;
  const int per = (B + kThreads - 1) / kThreads;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  long long local = 0;
  for (int b = b0; b < b1; ++b) local += kPieceCost + blocks_of(seq_len_of(p, b));
  local *= per_seq;
  long long incl = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) ctl->warp_sum[warp] = incl;
  __syncthreads();
  long long total = 0, run = incl - local;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) run += ctl->warp_sum[w];
    total += ctl->warp_sum[w];
  }
  const int parts = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  const int self = static_cast<int>(blockIdx.x);
  const long long chunk = divide(total, parts);
  const int extra = static_cast<int>(total - chunk * parts);
  const long long a0 = self * chunk + min(self, extra);
  if (self >= parts) {
    if (tid == 0) ctl->share = Share{0, 0, 0, 1, 0, 0, parts, 0};
  } else if (a0 >= run && a0 < run + local) {
    int b = b0;
    long long cost = 0;
    for (;; ++b) {  // ends: a0 lies in this thread's sequences
      cost = kPieceCost + blocks_of(seq_len_of(p, b));
      if (a0 < run + cost * per_seq) break;
      run += cost * per_seq;
    }
    const int entry = static_cast<int>(divide(a0 - run, static_cast<int>(cost)));
    ctl->share = Share{a0, a0 + chunk + (self < extra ? 1 : 0), run + entry * cost, chunk,
                       b, entry, parts, extra};
  }
  __syncthreads();
}

// A run of one entry's 64-token blocks.
struct Piece {
  int b, entry;    // entry of the sequence: kv head * head tiles + head tile
  int len, j0, nb; // tokens; first block; blocks of the entry
  int blocks;      // of the piece
  int n;           // this warp's 16-token tiles
  long long x;     // first unit of the entry
};

// Operand pair k (0..3) of w: nibble k of both 16-bit halves as f16 numbers c *
// 2^-24 (k even) or 16 c * 2^-24 (k odd); w8 = w >> 8.
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t w8, int k) {
  return (k < 2 ? w : w8) & ((k & 1) ? 0x00f000f0u : 0x000f000fu);
}
// The same with every code at bits 4 to 7 of its half: 16 c * 2^-24.
__device__ __forceinline__ uint32_t high_pair(uint32_t w, uint32_t w8, int k) {
  return (k == 0 ? w << 4 : k == 1 ? w : k == 2 ? w >> 4 : w8) & 0x00f000f0u;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Exponent field of |x| unbiased (-127 for zero and subnormals, 128 for an
// infinity), and 2^e for -126 <= e <= 127.
__device__ __forceinline__ int exponent_of(float x) {
  return static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// 8x8 transpose across the warp: lane l held row l / 4, columns 2 (l % 4), +1.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Cache words are read once: no L1 allocation.
template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t *src, uint32_t *w) {
  static_assert(kWords == 2 || kWords % 4 == 0, "vector width");
  if constexpr (kWords == 2)
    asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];"
                 : "=r"(w[0]), "=r"(w[1])
                 : "l"(src));
  else
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i)
      asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                   : "l"(src + 16 * i));
}
// A (lo, scale) pair of the cache.
template <typename T>
__device__ __forceinline__ void pair_of(uint32_t w, float &lo, float &scale) {
  const T *e = reinterpret_cast<const T *>(&w);
  lo = Elem<T>::to_f(e[0]);
  scale = Elem<T>::to_f(e[1]);
}

template <typename T, int kD, int kGroups, int kNT>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(kD, kNT))
    kv4_decode_kernel(const __grid_constant__ Params p) {
  using PL = Plan<kD, kGroups, kNT>;
  constexpr int kG = kD / kGroups;
  constexpr int kW = kD / 32;   // key words of a lane and token
  constexpr int kU = kD / 64;   // value words of a lane and token
  constexpr int kTileB = PL::kTileB, kHeads = PL::kHeads;
  constexpr bool kSplitP = std::is_same<T, __half>::value;
  constexpr bool kHighKeys = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Control ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  compute_share(p, &ctl);
  const Share &sh = ctl.share;
  float *obuf = reinterpret_cast<float *>(smem);
  float *kept = obuf + warp * kHeads * PL::kORow + lane;  // value sums of earlier tiles

  const int self = static_cast<int>(blockIdx.x), per_seq = p.hkv * p.head_tiles;
  // the next piece of the share, from the entry at unit x on
  int b = sh.b, entry = sh.entry, len = sh.a0 < sh.a1 ? seq_len_of(p, b) : 0;
  long long x = sh.x;
  auto next_piece = [&](Piece &pc) -> bool {
    while (x < sh.a1) {
      const int nb = blocks_of(len);
      // block j of the entry is unit x + kPieceCost + j
      const long long from = sh.a0 - x - kPieceCost, to = sh.a1 - x - kPieceCost;
      pc.j0 = static_cast<int>(min(max(from, 0ll), static_cast<long long>(nb)));
      pc.blocks = static_cast<int>(min(max(to, 0ll), static_cast<long long>(nb))) - pc.j0;
      pc.b = b;
      pc.entry = entry;
      pc.len = len;
      pc.nb = nb;
      pc.x = x;
      // an empty entry goes to the CTA that holds its first unit
      const bool mine = nb > 0 ? pc.blocks > 0 : x >= sh.a0;
      x += kPieceCost + nb;
      if (++entry == per_seq) {
        entry = 0;
        if (++b < p.batch) len = seq_len_of(p, b);
      }
      if (mine) {
        // block j holds this warp's tile j * 4 + warp
        const int tiles = (pc.len + kTileTokens - 1) / kTileTokens;
        pc.n = min(pc.blocks, max((tiles - warp + kWarps - 1) / kWarps - pc.j0, 0));
        return true;
      }
    }
    return false;
  };

  constexpr int kLaneWords = kW < 4 ? kW : 4;
  constexpr int kRowBytes = 16 * kLaneWords;
  const int key_off = r * kRowBytes + q * 4 * kLaneWords;  // row r + 8: + 8 * kRowBytes
  const int tiles_per_page = p.pool.tiles_per_block;
  uint32_t ka[kW] = {}, kb[kW] = {}, sca[2 * kGroups] = {}, scb[2 * kGroups] = {}, vw[4 * kU] = {};
  auto load_keys = [&](const uint8_t *tile) {
#pragma unroll
    for (int pl = 0; pl < kW / kLaneWords; ++pl) {
      const uint8_t *plane = tile + pl * (kTileTokens * kRowBytes) + key_off;
      load_words<kLaneWords>(plane, ka + pl * kLaneWords);
      load_words<kLaneWords>(plane + 8 * kRowBytes, kb + pl * kLaneWords);
    }
  };
  auto load_scales = [&](const uint8_t *tile) {  // all pairs of tokens r, r + 8
    load_words<2 * kGroups>(tile + 2 * code_bytes(kD) + r * 8 * kGroups, sca);
    load_words<2 * kGroups>(tile + 2 * code_bytes(kD) + (r + 8) * 8 * kGroups, scb);
  };
  auto load_values = [&](const uint8_t *tile) {  // [token pair][u][half]
#pragma unroll
    for (int pl = 0; pl < kU; ++pl)
      load_words<4>(tile + code_bytes(kD) + pl * 512 + lane * 16, vw + 4 * pl);
  };
  // every 32 tiles lane i looks up the pool tile of the warp's i-th next one
  // (-1: past the end, or a block outside the pool), one batch ahead
  auto look_up = [&](const Piece &pc, int i0) {
    const int mine = (pc.j0 + i0 + lane) * kWarps + warp;
    if (i0 + lane >= pc.n) return -1;
    const int pg = mine / tiles_per_page;
    const int page = __ldg(p.block_table + pc.b * p.bt_stride + pg);
    if (page < 0 || page >= p.num_blocks) return -1;
    return (page * p.hkv + pc.entry / p.head_tiles) * tiles_per_page + (mine - pg * tiles_per_page);
  };
  int tiles_a = -1, tiles_b = -1;  // tiles base .. + 31, + 32 .. + 63 of the piece
  auto tile_at = [&](int i) {      // i: relative to base, 0 .. 63
    return __shfl_sync(0xffffffffu, i < 32 ? tiles_a : tiles_b, i & 31);
  };
  auto tile_ptr = [&](int at) { return p.pool.data + static_cast<int64_t>(at) * kTileB; };
  auto prefetch = [&](int at) {
    if (at >= 0 && lane == 0) bulk_prefetch_l2(tile_ptr(at), kTileB);
  };
  // a piece's loads: Q rows, block table, its first tile into registers, the
  // next ones into L2.  Issued after the previous piece is merged (before, the
  // registers of both spill).
  uint4 qraw[kNT][kW];
  int at = -1;
  auto begin = [&](const Piece &pc) {
    const int h0 = pc.entry % p.head_tiles * kHeads;  // first head inside the group
    const int heads = min(kHeads, p.group - h0);
    const T *rows = static_cast<const T *>(p.q) + pc.b * p.q_sb +
                    static_cast<int64_t>(pc.entry / p.head_tiles * p.group + h0) * p.q_sh;
#pragma unroll
    for (int t = 0; t < kNT; ++t)
#pragma unroll
      for (int i = 0; i < kW; ++i)
        qraw[t][i] = t * 8 + r < heads
                         ? __ldg(reinterpret_cast<const uint4 *>(rows + (t * 8 + r) * p.q_sh) + 4 * i + q)
                         : make_uint4(0u, 0u, 0u, 0u);
    tiles_a = look_up(pc, 0);
    tiles_b = pc.n > 32 ? look_up(pc, 32) : -1;
    at = tile_at(0);
    if (at >= 0) {
      load_keys(tile_ptr(at));
      load_scales(tile_ptr(at));
      load_values(tile_ptr(at));
    }
#pragma unroll 1
    for (int i = 1; i < min(kAhead, pc.n); ++i) prefetch(tile_at(i));
  };

  Piece pc;
  bool have = next_piece(pc);
  if (have) begin(pc);
  while (have) {
    // Q as the B operand, times a power of two that brings the row's largest
    // magnitude to [2^13, 2^14): pair k of word i holds dims 32 i + 8 q + {k,
    // k + 4} of head r of each 8-head tile, over 16 for odd k
    uint32_t qf[kNT][kW][4];
    float qs[kNT][kGroups][2];  // 2^-24 * sum of q' over a group, heads 2 q, 2 q + 1
    float unit[kNT][2];         // log2 score per unit of the products' sum, ditto
#pragma unroll
    for (int t = 0; t < kNT; ++t) {
      float mag = 0.f;
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        const T *el = reinterpret_cast<const T *>(&qraw[t][i]);
#pragma unroll
        for (int d = 0; d < 8; ++d) mag = fmaxf(mag, fabsf(Elem<T>::to_f(el[d])));
      }
      mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
      mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
      const int f = max(exponent_of(mag) - 13, -100);
      const float norm = pow2(-f);
      float sum[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) sum[g] = 0.f;
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        const T *el = reinterpret_cast<const T *>(&qraw[t][i]);
        float x[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          x[d] = Elem<T>::to_f(el[d]) * norm;
          sum[32 * i / kG] += x[d];
        }
        constexpr float kOdd = kHighKeys ? 1.f : 0.0625f;
        qf[t][i][0] = Elem<__half>::pack2(x[0], x[4]);
        qf[t][i][1] = Elem<__half>::pack2(x[1] * kOdd, x[5] * kOdd);
        qf[t][i][2] = Elem<__half>::pack2(x[2], x[6]);
        qf[t][i][3] = Elem<__half>::pack2(x[3] * kOdd, x[7] * kOdd);
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        sum[g] *= kHighKeys ? 0x1p-20f : 0x1p-24f;
        qs[t][g][0] = __shfl_sync(0xffffffffu, sum[g], 8 * q);
        qs[t][g][1] = __shfl_sync(0xffffffffu, sum[g], 8 * q + 4);
      }
      // scale * 2^(f + 24), or 2^(f + 20)
      const float un = p.scale_log2 * pow2(f + 12) * (kHighKeys ? 256.f : 4096.f);
      unit[t][0] = __shfl_sync(0xffffffffu, un, 8 * q);
      unit[t][1] = __shfl_sync(0xffffffffu, un, 8 * q + 4);
    }

    // running state; lanes of equal q agree on m; l and extra are partial sums
    // over the lane's tokens; pu: P' per p * s, a power of two
    float o[kNT][kD / 16][4];
    uint64_t pu[kNT][kGroups], m[kNT], l[kNT], extra[kNT][kGroups];  // heads 2 q, 2 q + 1
    float limit[kGroups];  // of value scales: 2^kLimitTop over the lane's largest unit
#pragma unroll
    for (int g = 0; g < kGroups; ++g) limit[g] = 0.f;
#pragma unroll
    for (int t = 0; t < kNT; ++t) {
      m[t] = f32x2(kNoMax, kNoMax);
      l[t] = 0u;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        extra[t][g] = 0u;
        pu[t][g] = f32x2(pow2(kUnitMost), pow2(kUnitMost));
      }
#pragma unroll
      for (int i = 0; i < kD / 16; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[t][i][c] = 0.f;
    }

    // The tile's words are in registers; each set of them is loaded again, for
    // the warp's next tile, as soon as its products are issued.
    int base = 0;  // of tiles_a
#pragma unroll 1
    for (int i = 0; i < pc.n; ++i) {
      const int left = at >= 0 ? pc.len - ((pc.j0 + i) * kWarps + warp) * kTileTokens : 0;
      if (i - base == 32) {
        // The tensor cores cut off what an f32 sum has no room for, and the
        // codes' sums only grow (no sign): after 64 tiles they move to this
        // warp's part of the buffer, where they are added with rounding.
        if (base & 32) {
#pragma unroll
          for (int t = 0; t < kNT; ++t)
#pragma unroll
            for (int i2 = 0; i2 < kD / 16; ++i2)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float &sum = kept[((t * (kD / 16) + i2) * 4 + c) * 32];
                sum = base >= 64 ? sum + o[t][i2][c] : o[t][i2][c];
                o[t][i2][c] = 0.f;
              }
        }
        base += 32;
        tiles_a = tiles_b;
        tiles_b = base + 32 < pc.n ? look_up(pc, base + 32) : -1;
      }
      at = tile_at(i + 1 - base);
      prefetch(tile_at(i + kAhead - base));
      const uint8_t *next = tile_ptr(at);
      // ------------------------------------------------------------ scores
      float s[kNT][4];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        float acc[kNT][4];
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[t][c] = 0.f;
#pragma unroll
        for (int i2 = g * kW / kGroups; i2 < (g + 1) * kW / kGroups; ++i2) {
          const uint32_t ka8 = ka[i2] >> 8, kb8 = kb[i2] >> 8;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            auto key_pair = [](uint32_t w, uint32_t w8, int k) {
              return kHighKeys ? high_pair(w, w8, k) : code_pair(w, w8, k);
            };
            const uint32_t a0 = key_pair(ka[i2], ka8, 2 * ks), a1 = key_pair(kb[i2], kb8, 2 * ks),
                           a2 = key_pair(ka[i2], ka8, 2 * ks + 1),
                           a3 = key_pair(kb[i2], kb8, 2 * ks + 1);
#pragma unroll
            for (int t = 0; t < kNT; ++t)
              mma16816(acc[t], a0, a1, a2, a3, qf[t][i2][2 * ks], qf[t][i2][2 * ks + 1]);
          }
        }
        float loa, sa, lob, sb;
        pair_of<T>(sca[g], loa, sa);
        pair_of<T>(scb[g], lob, sb);
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[t][h] = fmaf(sa, acc[t][h], g == 0 ? loa * qs[t][g][h]
                                                 : fmaf(loa, qs[t][g][h], s[t][h]));
            s[t][h + 2] = fmaf(sb, acc[t][h + 2], g == 0 ? lob * qs[t][g][h]
                                                         : fmaf(lob, qs[t][g][h], s[t][h + 2]));
          }
      }
      if (at >= 0) load_keys(next);
#pragma unroll
      for (int t = 0; t < kNT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[t][c] *= unit[t][c & 1];
      if (left < kTileTokens) {  // tokens past the end: any bits, so select
        const bool la = r < left, lb = r + 8 < left;
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[t][h] = la ? s[t][h] : -INFINITY;
            s[t][h + 2] = lb ? s[t][h + 2] : -INFINITY;
          }
#pragma unroll
        for (int g = kGroups; g < 2 * kGroups; ++g) {
          sca[g] = la ? sca[g] : 0u;
          scb[g] = lb ? scb[g] : 0u;
        }
      }
      // --------------------------------------------------- running softmax
      uint64_t pa[kNT], pb[kNT];  // p of tokens r and r + 8
      auto weights = [&](int t) {
        float m0, m1;
        f32x2_split(m[t], m0, m1);
        pa[t] = f32x2(fast_exp2(s[t][0] - m0), fast_exp2(s[t][1] - m1));
        pb[t] = f32x2(fast_exp2(s[t][2] - m0), fast_exp2(s[t][3] - m1));
      };
      float top = -INFINITY;  // excess over the maxima
      bool over = false;      // a value scale past its limit
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        float m0, m1;
        f32x2_split(m[t], m0, m1);
        top = fmax3(top, fmaxf(s[t][0], s[t][2]) - m0, fmaxf(s[t][1], s[t][3]) - m1);
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        float lo, sa, sb;
        pair_of<T>(sca[kGroups + g], lo, sa);
        pair_of<T>(scb[kGroups + g], lo, sb);
        over |= fmaxf(sa, sb) > limit[g];
      }
      if (__any_sync(0xffffffffu, over || top > kRescaleThreshold)) {
        // Maxima are whole numbers: held sums move by powers of two, and a unit
        // stays that of the largest product met, in this tile or before.
        float most[kGroups];  // the lane's largest units
#pragma unroll
        for (int g = 0; g < kGroups; ++g) most[g] = 0.f;
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
          float mh[2], up[2], alpha[2];  // 2^n and 2^-n where the maximum grows by n
          f32x2_split(m[t], mh[0], mh[1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mx = fmaxf(s[t][h], s[t][h + 2]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1)
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float mn = fmaxf(mh[h], ceilf(mx));
            up[h] = pow2(static_cast<int>(fminf(mn - mh[h], 127.f)));
            alpha[h] = fast_exp2(mh[h] - mn);
            mh[h] = mn;
          }
          m[t] = f32x2(mh[0], mh[1]);
          weights(t);
          const uint64_t alpha2 = f32x2(alpha[0], alpha[1]);
          l[t] = fmul2(l[t], alpha2);
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            float lo, sa, sb, x0, x1, x2, x3, unit[2];
            pair_of<T>(sca[kGroups + g], lo, sa);
            pair_of<T>(scb[kGroups + g], lo, sb);
            f32x2_split(fmul2(pa[t], f32x2(sa, sa)), x0, x1);
            f32x2_split(fmul2(pb[t], f32x2(sb, sb)), x2, x3);
            // exponent fields (bias 127) of both heads' largest products
            uint32_t big = __float_as_uint(fmaxf(x0, x2)) >> 23 |
                           __float_as_uint(fmaxf(x1, x3)) >> 23 << 16;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1)
              big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, off));
            f32x2_split(pu[t][g], unit[0], unit[1]);
            extra[t][g] = fmul2(extra[t][g], alpha2);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int field = static_cast<int>(h ? big >> 16 : big & 0xffffu);
              const float now =
                  fminf(unit[h] * up[h], pow2(min(127 + kUnitTop - field, kUnitMost)));
              // 1 / 2^e: the exponent field mirrored about 127
              const float inv = __uint_as_float(0x7f000000u - __float_as_uint(unit[h]));
              const float held = alpha[h] * (now * inv);
              unit[h] = now;
              most[g] = fmaxf(most[g], now);
#pragma unroll
              for (int i2 = 0; i2 < kD / 16; ++i2) {
                if ((64 * (i2 / 4) + 32 * (i2 % 4 / 2)) / kG != g) continue;
                o[t][i2][h] *= held;
                o[t][i2][h + 2] *= held;
                if (base >= 64) {
                  kept[((t * (kD / 16) + i2) * 4 + h) * 32] *= held;
                  kept[((t * (kD / 16) + i2) * 4 + h + 2) * 32] *= held;
                }
              }
            }
            pu[t][g] = f32x2(unit[0], unit[1]);
          }
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          limit[g] = __uint_as_float(0x7f000000u + (kLimitTop << 23) - __float_as_uint(most[g]));
      }
      // ---------------------------------------------------------- P and P V
      uint32_t pf[kNT][kGroups][kSplitP ? 4 : 2];  // B operands (high, then low parts)
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        weights(t);
        l[t] = fadd2(l[t], fadd2(pa[t], pb[t]));
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float loa, sa, lob, sb, x0, x1, x2, x3;
          pair_of<T>(sca[kGroups + g], loa, sa);
          pair_of<T>(scb[kGroups + g], lob, sb);
          // in this order: p = 0 stays 0 whatever the unit and the scale
          f32x2_split(fmul2(fmul2(pa[t], pu[t][g]), f32x2(sa, sa)), x0, x1);
          f32x2_split(fmul2(fmul2(pb[t], pu[t][g]), f32x2(sb, sb)), x2, x3);
          const uint32_t wa = Elem<__half>::pack2(x0, x1), wb = Elem<__half>::pack2(x2, x3);
          pf[t][g][0] = transpose8(wa);
          pf[t][g][1] = transpose8(wb);
          if constexpr (kSplitP) {
            const __half2 ha = *reinterpret_cast<const __half2 *>(&wa);
            const __half2 hb = *reinterpret_cast<const __half2 *>(&wb);
            pf[t][g][2] = transpose8(Elem<__half>::pack2(x0 - __low2float(ha), x1 - __high2float(ha)));
            pf[t][g][3] = transpose8(Elem<__half>::pack2(x2 - __low2float(hb), x3 - __high2float(hb)));
          }
          extra[t][g] = ffma2(pa[t], f32x2(loa, loa), ffma2(pb[t], f32x2(lob, lob), extra[t][g]));
        }
      }
      if (at >= 0) load_scales(next);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const uint32_t w0 = vw[2 * u], w1 = vw[2 * u + 1], w2 = vw[2 * kU + 2 * u],
                       w3 = vw[2 * kU + 2 * u + 1];
        const uint32_t s0 = w0 >> 8, s1 = w1 >> 8, s2 = w2 >> 8, s3 = w3 >> 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int g = (64 * u + 32 * (k >> 1)) / kG;
          const uint32_t a0 = code_pair(w0, s0, k), a1 = code_pair(w1, s1, k),
                         a2 = code_pair(w2, s2, k), a3 = code_pair(w3, s3, k);
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
            mma16816(o[t][4 * u + k], a0, a1, a2, a3, pf[t][g][0], pf[t][g][1]);
            if constexpr (kSplitP)
              mma16816(o[t][4 * u + k], a0, a1, a2, a3, pf[t][g][2], pf[t][g][3]);
          }
        }
      }
      if (at >= 0) load_values(next);
    }

    if (base >= 64) {  // sums were moved
#pragma unroll
      for (int t = 0; t < kNT; ++t)
#pragma unroll
        for (int i2 = 0; i2 < kD / 16; ++i2)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[t][i2][c] += kept[((t * (kD / 16) + i2) * 4 + c) * 32];
      __syncwarp();  // the rows of the merge go over them
    }
    const Piece done = pc;

    // ------------------------------------------------ the warps' states meet
    const bool final_out = done.blocks == done.nb;
    const int h0 = done.entry % p.head_tiles * kHeads, kvh = done.entry / p.head_tiles;
    const int heads = min(kHeads, p.group - h0);
    const int slot = done.j0 == 0 ? sh.parts + self : self;
    if (done.j0 == 0 && threadIdx.x == 0) {
      int last = self;  // CTA with the entry's last block
      if (!final_out) {
        const long long u = done.x + kPieceCost + done.nb - 1, big = sh.extra * (sh.chunk + 1);
        last = static_cast<int>(u < big ? u / (sh.chunk + 1) : sh.extra + (u - big) / sh.chunk);
      }
      p.merge[static_cast<int64_t>(done.b) * per_seq + done.entry] =
          make_int4(final_out ? -1 : sh.parts + self, self + 1, last - self, 0);
    }
#pragma unroll
    for (int t = 0; t < kNT; ++t) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[t] = fadd2(l[t], __shfl_xor_sync(0xffffffffu, l[t], off));
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          extra[t][g] = fadd2(extra[t][g], __shfl_xor_sync(0xffffffffu, extra[t][g], off));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        auto of_head = [&](uint64_t x) {
          float x0, x1;
          f32x2_split(x, x0, x1);
          return h ? x1 : x0;
        };
        if (r == 0) {
          ctl.m[warp][t * 8 + 2 * q + h] = of_head(m[t]);
          ctl.l[warp][t * 8 + 2 * q + h] = of_head(l[t]);
        }
        float *row = obuf + (warp * kHeads + t * 8 + 2 * q + h) * PL::kORow;
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int pp = 0; pp < 2; ++pp) {
            const float ex = of_head(extra[t][(64 * u + 32 * pp) / kG]);
            const float inv = 1.f / of_head(pu[t][(64 * u + 32 * pp) / kG]);
            constexpr float even = 0x1p24f, odd = 0x1p20f;
            const float *oa = o[t][4 * u + 2 * pp], *ob = o[t][4 * u + 2 * pp + 1];
            // codes 2 pp and 2 pp + 1 of rows m < 8, then of rows m >= 8
            *reinterpret_cast<float4 *>(row + 64 * u + 32 * pp + 4 * r) =
                make_float4(fmaf(oa[h] * even, inv, ex), fmaf(ob[h] * odd, inv, ex),
                            fmaf(oa[h + 2] * even, inv, ex), fmaf(ob[h + 2] * odd, inv, ex));
          }
      }
    }
    __syncthreads();
    constexpr int kPer = kThreads / kHeads;       // threads of one head's row
    const int hh = threadIdx.x / kPer, part = threadIdx.x % kPer;
    float M = kNoMax;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ctl.m[w][hh]);
    float L = 0.f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = fast_exp2(ctl.m[w][hh] - M);
      L += ctl.l[w][hh] * f[w];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;  // a NaN stays one
    const float lse = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
    if (hh < heads) {
      const int h = kvh * p.group + h0 + hh;
      for (int d = part * 4; d < kD; d += kPer * 4) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4 *>(obuf + (w * kHeads + hh) * PL::kORow + d);
          const float k = f[w] * inv;
          acc.x = fmaf(v.x, k, acc.x);
          acc.y = fmaf(v.y, k, acc.y);
          acc.z = fmaf(v.z, k, acc.z);
          acc.w = fmaf(v.w, k, acc.w);
        }
        if (final_out)
          store4<T>(static_cast<T *>(p.o) + done.b * p.o_sb + h * p.o_sh + d, acc);
        else
          store4<float>(p.part_o + (static_cast<int64_t>(slot) * kHeads + hh) * kD + d, acc);
      }
      if (part == 0) {
        if (!final_out)  // the merge's maximum would drop a NaN: infinity keeps it
          p.part_lse[static_cast<int64_t>(slot) * kHeads + hh] = L == L ? lse : INFINITY;
        else if (p.lse)
          p.lse[static_cast<int64_t>(done.b) * p.hq + h] = lse;
      }
    }
    __syncthreads();  // the buffer is free for the next piece's sums
    have = next_piece(pc);
    if (have) begin(pc);
  }
}

// Merge of split entries: entry e = (sequence, kv head, run of head tiles),
// partials f32 [slot][rows][kD], o = sum_s exp(lse_s - lse) o_s.  What it costs is
// round trips to L2, so a warp loads eight partials of a row before it uses the
// first.  Narrow: one warp per row.  Wide, for entries cut into many pieces
// (one context of 8000 tokens: 74): eight warps per row take every eighth
// partial, and meet in shared memory.
template <typename T, int kD, bool kWide>
__global__ void __launch_bounds__(kWide ? 256 : 128)
    kv4_combine_kernel(const float *__restrict__ part_o, const float *__restrict__ part_lse,
                       const int4 *__restrict__ merge, int rows, int group, int head_tiles,
                       int hkv, int hq, T *__restrict__ out, int64_t o_sb, int64_t o_sh,
                       float *__restrict__ lse) {
  constexpr int kVec = kD > 128 ? 2 : 1, kAtOnce = 8, kRowWarps = kWide ? 8 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = kWide ? rows : rows / 4;  // blocks of an entry
  const int e = blockIdx.x / per, w = kWide ? warp : 0;
  const int row = kWide ? blockIdx.x % per : (blockIdx.x % per) * 4 + warp;
  const int ht = e % head_tiles, kvh = (e / head_tiles) % hkv, b = e / (head_tiles * hkv);
  const int in_group = ht * rows + row;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 mg = merge[e];
  if (mg.x < 0 || in_group >= group) return;  // of all threads when wide
  RowSum<kVec> st;
  st.init();
  st.template fold<kAtOnce>(part_o, part_lse, w, kRowWarps, 1 + mg.z, kD, lane, [&](int s) {
    return static_cast<int64_t>(s == 0 ? mg.x : mg.y + s - 1) * rows + row;
  });
  if constexpr (kWide) {
    __shared__ RowSum<kVec> states[kRowWarps][32];
    states[warp][lane] = st;
    __syncthreads();
    if (warp != 0) return;
    st.join(&states[0][lane], 32, kRowWarps);
  }
  const int h = kvh * group + in_group;
  const float l = st.finish(out + b * o_sb + h * o_sh, kD, lane);
  if (lse && lane == 0) lse[static_cast<int64_t>(b) * hq + h] = l;
}

// Run of query heads one entry serves, as 8-head tiles: two where a group has
// more than eight heads (the codes are expanded once for both), one for 256
// dims (two would not fit the registers).
int head_tiles_per_entry(int group, int d) { return group > 8 && d < 256 ? 2 : 1; }

template <typename T, int kD, int kGroups, int kNT>
int launch_t(const Params &p, int sms, cudaStream_t stream, int *grid_out, bool query) {
  using PL = Plan<kD, kGroups, kNT>;
  auto kern = kv4_decode_kernel<T, kD, kGroups, kNT>;
  *grid_out = sms * blocks_per_sm(kD, kNT);
  if (query) return FA_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(*grid_out);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = PL::kMergeBytes;  // below 48 KB: no opt-in needed
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  // about grid / entries pieces per entry; from 16 on the wide merge (8000 tokens
  // a context, 8 kv heads: 4 contexts 24.5 us wide, 26.6 narrow; 8 contexts 34.8 / 32.7)
  const int64_t entries = static_cast<int64_t>(p.batch) * p.hkv * p.head_tiles;
  const bool wide = entries * 16 <= *grid_out;
  const int64_t blocks = entries * (wide ? PL::kHeads : PL::kHeads / 4);
  if (blocks > INT32_MAX) return record_error(FA_ERR_UNSUPPORTED, "kv4 attention: too many rows");
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(wide ? 256 : 128);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg,
                         wide ? kv4_combine_kernel<T, kD, true> : kv4_combine_kernel<T, kD, false>,
                         static_cast<const float *>(p.part_o),
                         static_cast<const float *>(p.part_lse),
                         static_cast<const int4 *>(p.merge), PL::kHeads, p.group, p.head_tiles,
                         p.hkv, p.hq, static_cast<T *>(p.o), p.o_sb, p.o_sh, p.lse);
  if (e != cudaSuccess) return record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  return FA_OK;
}

template <typename T>
int launch_d(const fa_kv4_cache *c, const Params &p, int nt, int sms, cudaStream_t s, int *grid,
             bool query) {
  const int key = c->head_size * 10 + c->head_size / c->group_size;
  switch (key) {
    case 641: return nt == 2 ? launch_t<T, 64, 1, 2>(p, sms, s, grid, query) : launch_t<T, 64, 1, 1>(p, sms, s, grid, query);
    case 642: return nt == 2 ? launch_t<T, 64, 2, 2>(p, sms, s, grid, query) : launch_t<T, 64, 2, 1>(p, sms, s, grid, query);
    case 1281: return nt == 2 ? launch_t<T, 128, 1, 2>(p, sms, s, grid, query) : launch_t<T, 128, 1, 1>(p, sms, s, grid, query);
    case 1282: return nt == 2 ? launch_t<T, 128, 2, 2>(p, sms, s, grid, query) : launch_t<T, 128, 2, 1>(p, sms, s, grid, query);
    case 1284: return nt == 2 ? launch_t<T, 128, 4, 2>(p, sms, s, grid, query) : launch_t<T, 128, 4, 1>(p, sms, s, grid, query);
    case 2562: return launch_t<T, 256, 2, 1>(p, sms, s, grid, query);
    default: return launch_t<T, 256, 4, 1>(p, sms, s, grid, query);
  }
}

int validate_attention(const fa_kv4_attention_args *a) {
  if (!a) return record_error(FA_ERR_INVALID_ARGUMENT, "null args");
  const int st = validate_cache(&a->cache);
  if (st != FA_OK) return st;
  if (a->batch < 0 || a->num_q_heads <= 0 || a->num_q_heads % a->cache.num_kv_heads)
    return record_error(FA_ERR_INVALID_ARGUMENT,
                        "kv4 attention: query heads must be a multiple of the cache's kv heads");
  if (a->bt_width < 0 || a->bt_stride < 0)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4 attention: block table shape");
  if (!(a->scale > 0.f) || std::isinf(a->scale))
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4 attention: scale must be positive and finite");
  return FA_OK;
}

// Kernel parameters and grid; `query` leaves out the pointers' checks.
int run(const fa_kv4_attention_args *a, cudaStream_t stream, bool query, int *grid, int *entries,
        int *rows) {
  const int group = a->num_q_heads / a->cache.num_kv_heads;
  const int nt = head_tiles_per_entry(group, a->cache.head_size);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  Params p;
  p.q = a->q;
  p.q_sb = a->q_stride_b;
  p.q_sh = a->q_stride_h;
  p.pool = pool_of(&a->cache);
  p.num_blocks = a->cache.num_blocks;
  p.block_table = a->block_table;
  p.bt_stride = a->bt_stride;
  p.bt_width = a->bt_width;
  p.seq_lens = a->seq_lens;
  p.batch = a->batch;
  p.hq = a->num_q_heads;
  p.hkv = a->cache.num_kv_heads;
  p.group = group;
  p.head_tiles = (group + 8 * nt - 1) / (8 * nt);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.o = a->o;
  p.o_sb = a->o_stride_b;
  p.o_sh = a->o_stride_h;
  p.lse = a->lse;
  p.part_o = a->part_o;
  p.part_lse = a->part_lse;
  p.merge = reinterpret_cast<int4 *>(a->merge);
  *rows = 8 * nt;
  const int64_t n = static_cast<int64_t>(a->batch) * p.hkv * p.head_tiles;
  if (n > INT32_MAX / 16) return record_error(FA_ERR_UNSUPPORTED, "kv4 attention: too many rows");
  *entries = static_cast<int>(n);
  return a->cache.dtype == FA_DTYPE_F16
             ? launch_d<__half>(&a->cache, p, nt, sms, stream, grid, query)
             : launch_d<__nv_bfloat16>(&a->cache, p, nt, sms, stream, grid, query);
}

}  // namespace kv4
}  // namespace fa

extern "C" int fa_kv4_attention_workspace_size(const fa_kv4_attention_args *a, size_t *part_o_bytes,
                                               size_t *part_lse_bytes, size_t *merge_bytes) {
  using namespace fa::kv4;
  if (!part_o_bytes || !part_lse_bytes || !merge_bytes)
    return fa::record_error(FA_ERR_INVALID_ARGUMENT, "null out");
  int st = validate_attention(a);
  if (st != FA_OK) return st;
  int grid = 0, entries = 0, rows = 0;
  st = run(a, nullptr, true, &grid, &entries, &rows);
  if (st != FA_OK) return st;
  // two slots per CTA: its first and its last piece
  const size_t cells = 2 * static_cast<size_t>(grid) * rows;
  *part_o_bytes = cells * a->cache.head_size * sizeof(float);
  *part_lse_bytes = (cells * sizeof(float) + 15) / 16 * 16;
  *merge_bytes = static_cast<size_t>(entries) * 16;
  return FA_OK;
}

extern "C" int fa_kv4_attention(const fa_kv4_attention_args *a, void *stream) {
  using namespace fa::kv4;
  int st = validate_attention(a);
  if (st != FA_OK) return st;
  if (a->batch == 0) return FA_OK;
  auto al16 = [](const void *x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  if (!a->q || !a->o || !a->seq_lens || (!a->block_table && a->bt_width > 0) || !a->part_o ||
      !a->part_lse || !a->merge || (!a->cache.data && a->cache.num_blocks > 0))
    return fa::record_error(FA_ERR_INVALID_ARGUMENT, "kv4 attention: null tensor");
  if (!al16(a->q) || !al16(a->o) || !al16(a->part_o) || !al16(a->merge) || a->q_stride_b % 8 ||
      a->q_stride_h % 8 || a->o_stride_b % 8 || a->o_stride_h % 8)
    return fa::record_error(FA_ERR_INVALID_ARGUMENT,
                            "kv4 attention: q / o / workspace must be 16-byte aligned, strides "
                            "multiples of 8 elements");
  int grid = 0, entries = 0, rows = 0;
  return run(a, static_cast<cudaStream_t>(stream), false, &grid, &entries, &rows);
}
