// kv4_cache.cu -- write key / value rows to the 4-bit cache, read them back.
//
// A group of G dims of a row is held as its minimum lo, a scale s = (max -
// lo) / 15 rounded to the row's type (lo is an element of the row, so exact),
// and codes c = rint((x - lo) / s) clamped to 0 .. 15 (0 where s is 0); it
// stands for lo + s * c.  All arithmetic is f32 with IEEE division, so the
// result does not depend on the launch (reads: one fused
// multiply-add in the row's type, rounded once).  A group that holds a NaN or an
// infinity keeps lo = NaN and reads back as NaN: it is not lost silently.
//
// One segment of D / 8 lanes takes a token of one kv head, keys and values: a
// lane holds eight dims of each (two 16-byte loads), a group's minimum and
// maximum are shuffles inside the segment, and a lane's eight codes are one
// 32-bit word of keys and two 16-bit units of values (kv4.cuh).  4 D bytes in,
// D + 8 D / G out per token and head (the read in reverse).  At the HBM rate
// the schedulers have about 200 instructions per 16 elements of a lane, the
// integer pipes half of that, so per-element work is kept small: minima,
// maxima and expanded codes two at a time in T, divisions as products with the
// group's reciprocal corrected to the exact quotient, codes summed up as integers.
// A thread takes every grid-th token and loads the next ones' rows while it
// works on one; four blocks of 256 threads per SM.
//
// Measured: 16383 tokens of 8 kv heads of 128, groups of 64, bf16: 28.7 us to write
// (30.4 with a cold L2), 18.4 to read (20.4), 47.6 for both, 172 MB (3.6 TB/s).  Schedulers
// issue in 76% of the write's cycles and 59% of the read's, the integer pipe is
// 61% / 63% busy: the write is near its instruction count, the read waits.  64
// tokens: 6.1 us for both launches.
#include "kv4.cuh"
#include "flagattn_b200.h"

namespace fa {
int record_error(int status, const char *msg);  // capi.cu: message for fa_last_error()

namespace kv4 {

constexpr int kThreadsPerBlock = 256, kBlocksPerSm = 4;

struct RowsIn {
  const void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;  // elements
};
struct RowsOut {
  void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
};

// Elementwise minimum of two packed pairs that keeps a NaN.
template <typename T>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value)
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Tile and row of a pool slot; false for a slot outside the pool.
__device__ __forceinline__ bool find_slot(const Pool &pool, int64_t slot, int head, uint8_t *&tile,
                                          int &t) {
  if (static_cast<uint64_t>(slot) >= pool.slots) return false;  // negative ones too
  const uint32_t x = static_cast<uint32_t>(slot) / kTileTokens;
  const uint32_t block =
      static_cast<uint32_t>((static_cast<uint64_t>(x) * pool.div_mul) >> pool.div_shift);
  t = static_cast<int>(static_cast<uint32_t>(slot) % kTileTokens);
  tile = pool.tile(block, head, x - block * pool.tiles_per_block);
  return true;
}

// d / s correctly rounded, given r = 1 / s to about an ulp, for an s of at most
// 11 significant bits and results away from underflow: d * r is off by less
// than two ulp, and adding the exact remainder times r rounds a number that is
// off by 2^-22 ulp, while d / s is no nearer than 2^-12 ulp to a rounding boundary
// (it is a multiple of 2^-k / s, and no boundary: that has 25 significant bits).
// The method is Markstein's: one correction by the exact remainder.
__device__ __forceinline__ float quotient(float d, float s, float r) {
  const float q = d * r;
  return fmaf(fmaf(-q, s, d), r, q);
}
// 1 / s to about an ulp (one Newton step), s normal.
__device__ __forceinline__ float reciprocal(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return fmaf(fmaf(-s, r, 1.f), r, r);
}

// Codes of the lane's eight dims (u, 16 bits each), nibble i = dim i, and the
// group's (lo, scale) pair.  All lanes of the warp take part.
template <typename T, int kG>
__device__ __forceinline__ uint32_t quantise(const uint4 &u, uint32_t &pair) {
  constexpr int kLanes = kG / 8;  // of a group
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, half to even
  constexpr uint32_t kSigns = 0x80008000u;
  // {minimum, -maximum}: the minima of x and of -x
  const uint32_t lows = min2_nan<T>(min2_nan<T>(u.x, u.y), min2_nan<T>(u.z, u.w));
  const uint32_t highs = min2_nan<T>(min2_nan<T>(u.x ^ kSigns, u.y ^ kSigns),
                                     min2_nan<T>(u.z ^ kSigns, u.w ^ kSigns));
  uint32_t ends = min2_nan<T>(__byte_perm(lows, highs, 0x5410), __byte_perm(lows, highs, 0x7632));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1)
    ends = min2_nan<T>(ends, __shfl_xor_sync(0xffffffffu, ends, o));
  const T *end = reinterpret_cast<const T *>(&ends);
  const float lo = Elem<T>::to_f(end[0]), hi = -Elem<T>::to_f(end[1]);
  const bool finite = hi < INFINITY && lo > -INFINITY;  // false when a NaN came through
  // halves: max - min of finite bf16 values may pass the f32 range
  const float lo2 = lo * 0.5f, range2 = hi * 0.5f - lo2;
  const bool normal = range2 >= 0x1p-90f;
  const T scale =
      Elem<T>::from_f(normal ? quotient(range2, 7.5f, 1.f / 7.5f) : __fdiv_rn(range2, 7.5f));
  const float s2 = Elem<T>::to_f(scale) * 0.5f;
  T both[2] = {finite ? end[0] : Elem<T>::from_f(NAN), finite ? scale : Elem<T>::from_f(0.f)};
  pair = *reinterpret_cast<const uint32_t *>(both);
  if (!finite || s2 == 0.f) return 0u;
  const T *e = reinterpret_cast<const T *>(&u);
  // codes as integers in the mantissa of kMagic
  constexpr uint32_t kMagicBits = 0x4b400000u;
  uint32_t n[8];
  // Half of a scale that is normal in T (bf16: far above subnormal in f32 too).
  constexpr float kNormalHalf = std::is_same<T, __half>::value ? 0x1p-15f : 0x1p-100f;
  if (normal && s2 >= kNormalHalf) {
    // rint((x - lo) / s), at most 15: the scale is off by 2^-8 of itself at most
    const float r = reciprocal(s2);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      n[i] = __float_as_uint(quotient(fmaf(Elem<T>::to_f(e[i]), 0.5f, -lo2), s2, r) + kMagic);
  } else {  // a scale subnormal in T may be off by half: the quotient may pass 15
#pragma unroll
    for (int i = 0; i < 8; ++i)
      n[i] = __float_as_uint(
          fminf(__fdiv_rn(fmaf(Elem<T>::to_f(e[i]), 0.5f, -lo2), s2), 15.f) + kMagic);
  }
  // sum of 16^i (kMagicBits + code) modulo 2^32, less what kMagicBits gives
  uint32_t word = n[7];
#pragma unroll
  for (int i = 6; i >= 0; --i) word = word * 16u + n[i];
  return word - kMagicBits * 0x11111111u;
}

// kD dims, groups of kG.  Grid: token strides x kv heads; a segment takes every
// gridDim.x-th block's token and loads the next one's rows ahead.
template <typename T, int kD, int kG>
__global__ void __launch_bounds__(kThreadsPerBlock, kBlocksPerSm)
    append_kernel(RowsIn in, const int64_t *__restrict__ slots, int64_t n, Pool pool) {
  constexpr int kSeg = kD / 8, kGroups = kD / kG, kLanes = kG / 8, kTok = kThreadsPerBlock / kSeg;
  const int head = blockIdx.y, j = threadIdx.x % kSeg, r = j % 8, seg = threadIdx.x / kSeg;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTok;
  int64_t tok = static_cast<int64_t>(blockIdx.x) * kTok + seg;
  const T *k = static_cast<const T *>(in.k) + tok * in.k_st + head * in.k_sh + 8 * j;
  const T *v = static_cast<const T *>(in.v) + tok * in.v_st + head * in.v_sh + 8 * j;
  uint4 ku = make_uint4(0u, 0u, 0u, 0u), vu = ku;
  int64_t slot = -1;
  auto load = [&] {
    slot = -1;
    if (tok < n) {
      slot = __ldg(slots + tok);
      ku = __ldg(reinterpret_cast<const uint4 *>(k));
      vu = __ldg(reinterpret_cast<const uint4 *>(v));
    }
  };
  load();
  // all lanes of a warp stay while its first segment has a token
  for (int64_t first = tok - seg % (32 / kSeg); first < n; first += step) {
    const uint4 kc = ku, vc = vu;
    const int64_t at = slot;
    tok += step;
    k += step * in.k_st;
    v += step * in.v_st;
    load();
    uint32_t kpair, vpair;
    const uint32_t kword = quantise<T, kG>(kc, kpair), vword = quantise<T, kG>(vc, vpair);
    // the units (u, r, 0 / 1) gather four dims from each 32-dim half of their 64
    const uint32_t w0 = __shfl_sync(0xffffffffu, vword, (j & ~7) + r / 2, kSeg);
    const uint32_t w1 = __shfl_sync(0xffffffffu, vword, (j & ~7) + 4 + r / 2, kSeg);
    uint8_t *tile;
    int t;
    if (!find_slot(pool, at, head, tile, t)) continue;
    *reinterpret_cast<uint32_t *>(tile + key_word<kD>(t, j)) = kword;
    // byte `half` of the chosen 16-bit halves of w0, then of w1
    const uint32_t w = __byte_perm(w0, w1, (r & 1) ? 0x7362 : 0x5140);
#pragma unroll
    for (int half = 0; half < 2; ++half)
      *reinterpret_cast<uint16_t *>(tile + code_bytes(kD) + value_unit<kD>(t, j / 8, r, half)) =
          static_cast<uint16_t>(w >> (16 * half));
    if (j % kLanes == 0) {
      uint32_t *pairs = reinterpret_cast<uint32_t *>(tile + 2 * code_bytes(kD) + t * (8 * kGroups));
      pairs[j / kLanes] = kpair;
      pairs[kGroups + j / kLanes] = vpair;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value)
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value)
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  else
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// Eight values lo + scale * code, rounded once to T: two at a time in T, whose
// fused multiply-add takes exact operands.  A code is one AND-OR into the
// mantissa of a power of two (128 in bf16, 1024 in f16), which is then taken off.
template <typename T>
__device__ __forceinline__ uint4 expand(uint32_t word, uint32_t pair) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr uint32_t kPower = kHalf ? 0x64006400u : 0x43004300u, kMinusPower = kPower | 0x80008000u;
  const uint32_t lo = __byte_perm(pair, 0u, 0x1010), s = __byte_perm(pair, 0u, 0x3232);
  uint32_t x[4];  // dims i and i + 4
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = fma2<T>(add2<T>(((word >> (4 * i)) & 0x000f000fu) | kPower, kMinusPower), s, lo);
  // lo + 15 * scale may pass the type's largest number by the scale's rounding
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = min2_nan<T>(x[i], kHalf ? 0x7bff7bffu : 0x7f7f7f7fu);
  return make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410),
                    __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
}

template <typename T, int kD, int kG>
__global__ void __launch_bounds__(kThreadsPerBlock, kBlocksPerSm)
    read_kernel(Pool pool, const int64_t *__restrict__ slots, int64_t n, RowsOut out) {
  constexpr int kSeg = kD / 8, kGroups = kD / kG, kLanes = kG / 8, kTok = kThreadsPerBlock / kSeg;
  const int head = blockIdx.y, j = threadIdx.x % kSeg, r = j % 8, seg = threadIdx.x / kSeg;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTok;
  int64_t tok = static_cast<int64_t>(blockIdx.x) * kTok + seg;
  T *k = static_cast<T *>(out.k) + tok * out.k_st + head * out.k_sh + 8 * j;
  T *v = static_cast<T *>(out.v) + tok * out.v_st + head * out.v_sh + 8 * j;
  int64_t slot = tok < n ? __ldg(slots + tok) : -1;
  uint32_t kword, kpair, vpair;
  uint16_t v0, v1;
  auto load = [&] {  // of `slot`; zeros for a slot outside the pool
    kword = kpair = vpair = 0u;
    v0 = v1 = 0;
    uint8_t *tile;
    int t;
    if (!find_slot(pool, slot, head, tile, t)) return;
    kword = *reinterpret_cast<const uint32_t *>(tile + key_word<kD>(t, j));
    const uint8_t *codes = tile + code_bytes(kD);
    v0 = *reinterpret_cast<const uint16_t *>(codes + value_unit<kD>(t, j / 8, r, 0));
    v1 = *reinterpret_cast<const uint16_t *>(codes + value_unit<kD>(t, j / 8, r, 1));
    const uint32_t *pairs =
        reinterpret_cast<const uint32_t *>(tile + 2 * code_bytes(kD) + t * (8 * kGroups));
    kpair = pairs[j / kLanes];
    vpair = pairs[kGroups + j / kLanes];
  };
  load();
  slot = tok + step < n ? __ldg(slots + tok + step) : -1;
  for (int64_t first = tok - seg % (32 / kSeg); first < n; first += step) {
    const uint32_t kw = kword, kp = kpair, vp = vpair, vword = v0 | static_cast<uint32_t>(v1) << 16;
    const bool live = tok < n;
    T *kd = k, *vd = v;
    tok += step;
    k += step * out.k_st;
    v += step * out.v_st;
    load();  // the next token's words, and the slot of the one after it
    slot = tok + step < n ? __ldg(slots + tok + step) : -1;
    // values: dims 8 j .. + 3 are one byte of both units of r = 2 (j % 4), the
    // next four of r + 1; the byte is the 32-dim half p = (j / 4) % 2
    const uint32_t w0 = __shfl_sync(0xffffffffu, vword, (j & ~7) + 2 * (j % 4), kSeg);
    const uint32_t w1 = __shfl_sync(0xffffffffu, vword, (j & ~7) + 2 * (j % 4) + 1, kSeg);
    if (!live) continue;
    *reinterpret_cast<uint4 *>(kd) = expand<T>(kw, kp);
    *reinterpret_cast<uint4 *>(vd) =
        expand<T>(__byte_perm(w0, w1, ((j >> 2) & 1) ? 0x7531 : 0x6420), vp);
  }
}

// Calls fn with (T, head size, group size) as types / constants of the cache.
template <typename Fn>
int dispatch(const fa_kv4_cache *c, Fn fn) {
  auto by_type = [&](auto d, auto g) {
    return c->dtype == FA_DTYPE_F16 ? fn(__half(), d, g) : fn(__nv_bfloat16(), d, g);
  };
  using std::integral_constant;
  const int key = c->head_size * 1000 + c->group_size;
  switch (key) {
    case 64032: return by_type(integral_constant<int, 64>(), integral_constant<int, 32>());
    case 64064: return by_type(integral_constant<int, 64>(), integral_constant<int, 64>());
    case 128032: return by_type(integral_constant<int, 128>(), integral_constant<int, 32>());
    case 128064: return by_type(integral_constant<int, 128>(), integral_constant<int, 64>());
    case 128128: return by_type(integral_constant<int, 128>(), integral_constant<int, 128>());
    case 256064: return by_type(integral_constant<int, 256>(), integral_constant<int, 64>());
    default: return by_type(integral_constant<int, 256>(), integral_constant<int, 128>());
  }
}

int validate_cache(const fa_kv4_cache *c) {
  if (!c) return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: null cache");
  if (c->dtype != FA_DTYPE_BF16 && c->dtype != FA_DTYPE_F16)
    return record_error(FA_ERR_UNSUPPORTED, "kv4: rows are bf16 or f16");
  const int d = c->head_size, g = c->group_size;
  if (!(d == 64 || d == 128 || d == 256))
    return record_error(FA_ERR_UNSUPPORTED, "kv4: head size must be 64, 128 or 256");
  if (!(g == 32 || g == 64 || g == 128) || g > d || d / g > 4)
    return record_error(FA_ERR_UNSUPPORTED,
                        "kv4: group size must be 32, 64 or 128, with 1 to 4 groups per head");
  if (c->num_blocks < 0 || c->num_kv_heads <= 0)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: block / head count");
  if (c->block_size <= 0 || c->block_size % kTileTokens)
    return record_error(FA_ERR_UNSUPPORTED, "kv4: block size must be a multiple of 16 tokens");
  const int64_t slots = static_cast<int64_t>(c->num_blocks) * c->block_size;
  if (slots > 0xffffffffll || slots / kTileTokens > 0x7fffffffll / c->num_kv_heads)
    return record_error(FA_ERR_UNSUPPORTED, "kv4: pool of 2^32 slots or 2^31 tiles");
  if (reinterpret_cast<uintptr_t>(c->data) & 15u)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: the pool must be 16-byte aligned");
  return FA_OK;
}

Pool pool_of(const fa_kv4_cache *c) {
  Pool p;
  p.data = static_cast<uint8_t *>(c->data);
  p.slots = static_cast<uint32_t>(static_cast<int64_t>(c->num_blocks) * c->block_size);
  p.block_size = c->block_size;
  p.tiles_per_block = c->block_size / kTileTokens;
  p.heads = c->num_kv_heads;
  p.tile_bytes = tile_bytes(c->head_size, c->head_size / c->group_size);
  // x < 2^28 and 2^(l - 1) < d <= 2^l: m = floor(2^(28 + l) / d) + 1 is below
  // 2^30 and x * m >> (28 + l) is x / d, since m d - 2^(28 + l) <= d <= 2^l
  uint32_t l = 0;
  while ((1u << l) < static_cast<uint32_t>(p.tiles_per_block)) ++l;
  p.div_shift = 28 + l;
  p.div_mul = static_cast<uint32_t>((uint64_t{1} << p.div_shift) / p.tiles_per_block + 1);
  return p;
}

// Checks and grid shared by append and read: rows in either direction.
int validate_rows(const fa_kv4_cache *c, const void *k, int64_t k_st, int64_t k_sh, const void *v,
                  int64_t v_st, int64_t v_sh, const int64_t *slots, int64_t n, dim3 *grid) {
  const int st = validate_cache(c);
  if (st != FA_OK) return st;
  *grid = dim3(0);
  if (n < 0) return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: negative row count");
  if (n == 0) return FA_OK;
  if (!k || !v || !slots || (!c->data && c->num_blocks > 0))
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: null pointer");
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) ||
      (reinterpret_cast<uintptr_t>(slots) & 7u))
    return record_error(FA_ERR_INVALID_ARGUMENT,
                        "kv4: rows must be 16-byte aligned, slots 8-byte aligned");
  if (k_st % 8 || k_sh % 8 || v_st % 8 || v_sh % 8)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: strides must be multiples of 8 elements");
  const int64_t per_block = kThreadsPerBlock / (c->head_size / 8);
  if (n > 0x7fffffffLL * per_block || c->num_kv_heads > 65535)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: too many rows or kv heads");
  // as many blocks as are resident at once: the rest of the tokens in strides
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  const int64_t most = (kBlocksPerSm * sms + c->num_kv_heads - 1) / c->num_kv_heads;
  const int64_t want = (n + per_block - 1) / per_block;
  *grid = dim3(static_cast<unsigned>(want < most ? want : most),
               static_cast<unsigned>(c->num_kv_heads));
  return FA_OK;
}

}  // namespace kv4
}  // namespace fa

extern "C" int fa_kv4_cache_bytes(const fa_kv4_cache *c, int64_t *bytes) {
  using namespace fa::kv4;
  const int st = validate_cache(c);
  if (st != FA_OK) return st;
  if (!bytes) return fa::record_error(FA_ERR_INVALID_ARGUMENT, "kv4: null out");
  int64_t n = 0;
  const int64_t tiles = c->block_size / kTileTokens;
  if (__builtin_mul_overflow(tiles * c->num_kv_heads, static_cast<int64_t>(c->num_blocks), &n) ||
      __builtin_mul_overflow(n, pool_of(c).tile_bytes, &n))
    return fa::record_error(FA_ERR_INVALID_ARGUMENT, "kv4: pool size overflows");
  *bytes = n;
  return FA_OK;
}

extern "C" int fa_kv4_append(const fa_kv4_cache *c, const void *k, int64_t k_stride_t,
                             int64_t k_stride_h, const void *v, int64_t v_stride_t,
                             int64_t v_stride_h, const int64_t *slots, int64_t n, void *stream) {
  using namespace fa::kv4;
  dim3 grid;
  const int st = validate_rows(c, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, slots, n,
                               &grid);
  if (st != FA_OK || grid.x == 0) return st;
  const RowsIn in{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  return dispatch(c, [&](auto t, auto d, auto g) {
    append_kernel<decltype(t), d.value, g.value>
        <<<grid, kThreadsPerBlock, 0, static_cast<cudaStream_t>(stream)>>>(in, slots, n,
                                                                            pool_of(c));
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FA_OK : fa::record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  });
}

extern "C" int fa_kv4_read(const fa_kv4_cache *c, void *k, int64_t k_stride_t, int64_t k_stride_h,
                           void *v, int64_t v_stride_t, int64_t v_stride_h, const int64_t *slots,
                           int64_t n, void *stream) {
  using namespace fa::kv4;
  dim3 grid;
  const int st = validate_rows(c, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, slots, n,
                               &grid);
  if (st != FA_OK || grid.x == 0) return st;
  const RowsOut out{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  return dispatch(c, [&](auto t, auto d, auto g) {
    read_kernel<decltype(t), d.value, g.value>
        <<<grid, kThreadsPerBlock, 0, static_cast<cudaStream_t>(stream)>>>(pool_of(c), slots,
                                                                            n, out);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FA_OK : fa::record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  });
}
