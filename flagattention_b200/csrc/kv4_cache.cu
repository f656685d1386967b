// kv4_cache.cu -- write key / value rows to the 4-bit cache, read them back.
//
// A group of G dims of a row is held as its minimum lo, a scale s = (max -
// lo) / 15 rounded to the row's type (lo is an element of the row, so exact),
// and codes c = rint((x - lo) / s) clamped to 0 .. 15 (0 where s is 0); it
// stands for lo + s * c.  All arithmetic is f32 with IEEE division, so the
// result does not depend on the launch.  A group that holds a NaN or an
// infinity keeps lo = NaN and reads back as NaN: it is not lost silently.
//
// One segment of D / 8 lanes takes one row (token, kv head, keys or values):
// a lane holds eight dims (one 16-byte load), a group's minimum and maximum
// are shuffles inside the segment, and a lane's eight codes are one 32-bit
// word of the tile (kv4.cuh).  Byte-bound: 2 D bytes of a row in, D / 2 + 4 D
// / G out.
#include "kv4.cuh"
#include "flagattn_b200.h"

namespace fa {
int record_error(int status, const char *msg);  // capi.cu: message for fa_last_error()

namespace kv4 {

constexpr int kWarpsPerBlock = 8;

struct RowsIn {
  const void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;  // elements
};
struct RowsOut {
  void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
};

// Row of the calling lane: segment of D / 8 lanes = (token, head, keys / values).
template <int kD>
__device__ __forceinline__ bool locate(int64_t n, int heads, int64_t &tok, int &head, int &is_v,
                                       int &j) {
  constexpr int kSeg = kD / 8;
  const int64_t thread = static_cast<int64_t>(blockIdx.x) * (32 * kWarpsPerBlock) + threadIdx.x;
  const int64_t row = thread / kSeg;
  j = static_cast<int>(thread % kSeg);
  is_v = static_cast<int>(row & 1);
  head = static_cast<int>((row >> 1) % heads);
  tok = (row >> 1) / heads;
  return tok < n;
}

// kD dims, groups of kG.
template <typename T, int kD, int kG>
__global__ void __launch_bounds__(32 * kWarpsPerBlock)
    append_kernel(RowsIn in, const int64_t *__restrict__ slots, int64_t n, Pool pool) {
  constexpr int kSeg = kD / 8, kGroups = kD / kG, kLanes = kG / 8;  // lanes of a group
  int64_t tok;
  int head, is_v, j;
  const bool inside = locate<kD>(n, pool.heads, tok, head, is_v, j);
  const int64_t slot = inside ? __ldg(slots + tok) : -1;
  const bool live = slot >= 0 && slot < pool.slots;
  float x[8];
  bool bad = false;
  float lo = INFINITY, hi = -INFINITY;
  if (live) {
    const T *src = is_v ? static_cast<const T *>(in.v) + tok * in.v_st + head * in.v_sh
                        : static_cast<const T *>(in.k) + tok * in.k_st + head * in.k_sh;
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(src) + j);
    const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = Elem<T>::to_f(e[i]);
      bad |= !(fabsf(x[i]) < INFINITY);
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad |= __shfl_xor_sync(0xffffffffu, static_cast<int>(bad), o) != 0;
  }
  // halves: max - min of finite bf16 values may pass the f32 range
  const T scale = Elem<T>::from_f(__fdiv_rn(hi * 0.5f - lo * 0.5f, 7.5f));
  const float s = Elem<T>::to_f(scale);
  uint32_t word = 0;
  if (!bad && s != 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = rintf(__fdiv_rn(x[i] * 0.5f - lo * 0.5f, s * 0.5f));
      word |= static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f)) << (4 * i);
    }
  }
  // the units (u, r, 0 / 1) gather four dims from each 32-dim half of their 64
  const int r = j % 8;
  const uint32_t w0 = __shfl_sync(0xffffffffu, word, (j & ~7) + r / 2, kSeg);
  const uint32_t w1 = __shfl_sync(0xffffffffu, word, (j & ~7) + 4 + r / 2, kSeg);
  if (!live) return;
  const int64_t block = slot / pool.block_size;
  const int off = static_cast<int>(slot % pool.block_size), t = off % kTileTokens;
  uint8_t *tile = pool.tile(block, head, off / kTileTokens);
  if (is_v) {  // byte `half` of the chosen 16-bit halves of w0, then of w1
    const uint32_t w = __byte_perm(w0, w1, (r & 1) ? 0x7362 : 0x5140);
#pragma unroll
    for (int half = 0; half < 2; ++half)
      *reinterpret_cast<uint16_t *>(tile + code_bytes(kD) + value_unit<kD>(t, j / 8, r, half)) =
          static_cast<uint16_t>(w >> (16 * half));
  } else {
    *reinterpret_cast<uint32_t *>(tile + key_word<kD>(t, j)) = word;
  }
  if (j % kLanes == 0) {
    T pair[2] = {bad ? Elem<T>::from_f(NAN) : Elem<T>::from_f(lo),
                 bad ? Elem<T>::from_f(0.f) : scale};
    *reinterpret_cast<uint32_t *>(tile + 2 * code_bytes(kD) + t * (8 * kGroups) +
                                  (is_v * kGroups + j / kLanes) * 4) =
        *reinterpret_cast<const uint32_t *>(pair);
  }
}

template <typename T, int kD, int kG>
__global__ void __launch_bounds__(32 * kWarpsPerBlock)
    read_kernel(Pool pool, const int64_t *__restrict__ slots, int64_t n, RowsOut out) {
  constexpr int kSeg = kD / 8, kGroups = kD / kG, kLanes = kG / 8;
  int64_t tok;
  int head, is_v, j;
  const bool inside = locate<kD>(n, pool.heads, tok, head, is_v, j);
  const int64_t slot = inside ? __ldg(slots + tok) : -1;
  const bool live = slot >= 0 && slot < pool.slots;
  uint32_t word = 0;
  float lo = 0.f, s = 0.f;
  const int r = j % 8;
  if (live) {
    const int64_t block = slot / pool.block_size;
    const int off = static_cast<int>(slot % pool.block_size), t = off % kTileTokens;
    const uint8_t *tile = pool.tile(block, head, off / kTileTokens);
    if (is_v) {
      const uint8_t *codes = tile + code_bytes(kD);
      word = *reinterpret_cast<const uint16_t *>(codes + value_unit<kD>(t, j / 8, r, 0)) |
             static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(
                 codes + value_unit<kD>(t, j / 8, r, 1))) << 16;
    } else {
      word = *reinterpret_cast<const uint32_t *>(tile + key_word<kD>(t, j));
    }
    const uint32_t pair = *reinterpret_cast<const uint32_t *>(
        tile + 2 * code_bytes(kD) + t * (8 * kGroups) + (is_v * kGroups + j / kLanes) * 4);
    const T *e = reinterpret_cast<const T *>(&pair);
    lo = Elem<T>::to_f(e[0]);
    s = Elem<T>::to_f(e[1]);
  }
  // values: dims 8 j .. + 3 are one byte of both units of r = 2 (j % 4), the
  // next four of r + 1; the byte is the 32-dim half p = (j / 4) % 2
  const uint32_t w0 = __shfl_sync(0xffffffffu, word, (j & ~7) + 2 * (j % 4), kSeg);
  const uint32_t w1 = __shfl_sync(0xffffffffu, word, (j & ~7) + 2 * (j % 4) + 1, kSeg);
  if (!inside) return;
  if (is_v) word = __byte_perm(w0, w1, ((j >> 2) & 1) ? 0x7531 : 0x6420);
  // lo + 15 * scale may pass the type's largest number by the scale's rounding
  const float top = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
  auto value = [&](int i) {
    const float x = fmaf(static_cast<float>((word >> (4 * i)) & 15u), s, lo);
    return x > top ? top : x;  // false for a NaN
  };
  uint4 u;
  uint32_t *o = reinterpret_cast<uint32_t *>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = Elem<T>::pack2(value(2 * i), value(2 * i + 1));
  T *dst = is_v ? static_cast<T *>(out.v) + tok * out.v_st + head * out.v_sh
                : static_cast<T *>(out.k) + tok * out.k_st + head * out.k_sh;
  reinterpret_cast<uint4 *>(dst)[j] = u;
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
  if (reinterpret_cast<uintptr_t>(c->data) & 15u)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: the pool must be 16-byte aligned");
  return FA_OK;
}

Pool pool_of(const fa_kv4_cache *c) {
  Pool p;
  p.data = static_cast<uint8_t *>(c->data);
  p.slots = static_cast<int64_t>(c->num_blocks) * c->block_size;
  p.block_size = c->block_size;
  p.heads = c->num_kv_heads;
  p.tile_bytes = tile_bytes(c->head_size, c->head_size / c->group_size);
  return p;
}

// Checks and grid shared by append and read: rows in either direction.
int validate_rows(const fa_kv4_cache *c, const void *k, int64_t k_st, int64_t k_sh, const void *v,
                  int64_t v_st, int64_t v_sh, const int64_t *slots, int64_t n, unsigned *grid) {
  const int st = validate_cache(c);
  if (st != FA_OK) return st;
  *grid = 0;
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
  const int64_t per_block = 32 * kWarpsPerBlock / (c->head_size / 8);
  if (n > (int64_t{1} << 40) / c->num_kv_heads)
    return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: too many rows");
  const int64_t blocks = (n * c->num_kv_heads * 2 + per_block - 1) / per_block;
  if (blocks > 0x7fffffffLL) return record_error(FA_ERR_INVALID_ARGUMENT, "kv4: too many rows");
  *grid = static_cast<unsigned>(blocks);
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
  unsigned grid = 0;
  const int st = validate_rows(c, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, slots, n,
                               &grid);
  if (st != FA_OK || grid == 0) return st;
  const RowsIn in{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  return dispatch(c, [&](auto t, auto d, auto g) {
    append_kernel<decltype(t), d.value, g.value>
        <<<grid, 32 * kWarpsPerBlock, 0, static_cast<cudaStream_t>(stream)>>>(in, slots, n,
                                                                            pool_of(c));
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FA_OK : fa::record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  });
}

extern "C" int fa_kv4_read(const fa_kv4_cache *c, void *k, int64_t k_stride_t, int64_t k_stride_h,
                           void *v, int64_t v_stride_t, int64_t v_stride_h, const int64_t *slots,
                           int64_t n, void *stream) {
  using namespace fa::kv4;
  unsigned grid = 0;
  const int st = validate_rows(c, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, slots, n,
                               &grid);
  if (st != FA_OK || grid == 0) return st;
  const RowsOut out{k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h};
  return dispatch(c, [&](auto t, auto d, auto g) {
    read_kernel<decltype(t), d.value, g.value>
        <<<grid, 32 * kWarpsPerBlock, 0, static_cast<cudaStream_t>(stream)>>>(pool_of(c), slots,
                                                                            n, out);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FA_OK : fa::record_error(FA_ERR_CUDA, cudaGetErrorString(e));
  });
}
