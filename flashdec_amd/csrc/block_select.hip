// Blocks that matter to a query, by a cheap score, for gfx950.
//
//   bounds: of a block's keys, the least lo_d and the largest hi_d in every dim.
//   select: for queries q of the heads that share a KV head,
//             s(block) = sum_heads sum_d max(q_d lo_d, q_d hi_d)
//           is at least the sum of the heads' products with any key of the block.  As
//           max(q lo, q hi) = max(q, 0) hi + min(q, 0) lo, the heads add up first:
//             s = sum_d Qp_d hi_d + Qm_d lo_d,  Qp = sum max(q, 0), Qm = sum min(q, 0),
//           2 D products a block, however many heads there are.
//
// The sum is taken in 64 bits and rounded once to 32, so that the order in which it
// is added does not decide between blocks: products of 16-bit numbers and a sum of a
// few hundred of them err there far below a 32-bit step.
#include <type_traits>

#include "decode_host.h"
#include "fp4_format.h"

namespace fd {

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// ============================================================= bounds ====
struct BoundsParams {
  const void* k;
  int64_t ks0, ks1, ks2, ks3;
  const void* bt;
  int64_t bts0, bts1;
  const void* sl;
  int64_t sls;
  void* bounds;  // [block, head, 2, D], contiguous
  int bt_i64, sl_i64, hkv, head_dim, block_size, width;
  int64_t num_blocks, new_tokens;
};

// 16-bit floating-point numbers as whole numbers of the same order, two a word (its own
// inverse): NaN lie beyond the infinities, at the end of their sign.
__device__ __forceinline__ uint32_t ordered16(uint32_t x) {
  const s16x2 sign = __builtin_bit_cast(s16x2, x) >> 15;
  return x ^ (__builtin_bit_cast(uint32_t, sign) & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t min16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
__device__ __forceinline__ uint32_t max16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}

// Bounds of a dim whose least and largest number, so ordered, these are: NaN where one
// of them is.
template <typename T>
__device__ __forceinline__ void bounds_of(uint32_t& lo, uint32_t& hi) {
  constexpr int kInf = std::is_same_v<T, __bf16> ? 0x7f80 : 0x7c00;
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = static_cast<int16_t>(lo >> (16 * e)), y = static_cast<int16_t>(hi >> (16 * e));
    const bool odd = x < ~kInf || y > kInf;  // (~code: the negative number of that magnitude)
    a |= (odd ? 0x7fffu : ordered16(static_cast<uint16_t>(x)) & 0xffffu) << (16 * e);
    b |= (odd ? 0x7fffu : ordered16(static_cast<uint16_t>(y)) & 0xffffu) << (16 * e);
  }
  lo = a;
  hi = b;
}

// The row's i-th block with new tokens, or -1 where that is not complete or not in the
// pool.
__device__ __forceinline__ int64_t fresh_block(const BoundsParams& p, int b, int64_t i) {
  const int64_t cap = static_cast<int64_t>(p.width) * p.block_size;
  int64_t len = load_index_uniform(p.sl, b * p.sls, p.sl_i64);
  len = len < 0 ? 0 : (len < cap ? len : cap);
  const int64_t first = (len > p.new_tokens ? len - p.new_tokens : 0) / p.block_size;
  if (first + i >= len / p.block_size) return -1;
  BlockId id = load_block_id_uniform(p.bt, b * p.bts0 + (first + i) * p.bts1, p.bt_i64);
  if (!p.bt_i64) id.high = 0;
  return id.below(p.num_blocks) ? id.low : -1;
}

constexpr int kBoundsWaves = 4;

// Least and largest of x[0 .. N) of every lane and of the lanes L apart, as bounds.
template <typename T, int L, int N>
__device__ __forceinline__ void reduce_bounds(const uint32_t (&x)[N], uint32_t& lo, uint32_t& hi) {
  lo = hi = ordered16(x[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) {
    const uint32_t y = ordered16(x[i]);
    lo = min16(lo, y);
    hi = max16(hi, y);
  }
#pragma unroll
  for (int o = 32; o >= L; o >>= 1) {
    lo = min16(lo, static_cast<uint32_t>(__shfl_xor(static_cast<int>(lo), o, 64)));
    hi = max16(hi, static_cast<uint32_t>(__shfl_xor(static_cast<int>(hi), o, 64)));
  }
  bounds_of<T>(lo, hi);
}

// Rows of 16-byte pieces: a wave a (block, head), D / 8 lanes a token, BS / (512 / D)
// loads a lane, all on their way at once.  Whole numbers take 2.5 instructions an
// element, two at a time; bound by the read (four rows of 16384 .. 32768 tokens, Hkv 8,
// D 128: 214 MB in 39 us, 5.5 TB/s, from a warm last-level cache 32; a thread a dim took
// 82).  The loads leave the caches to others (47.3 -> 41.9 us a call).
template <typename T, int BS, int D>
__global__ __launch_bounds__(64 * kBoundsWaves) void key_bounds_rows_kernel(BoundsParams p) {
  constexpr int L = D / 8, G = 64 / L, N = BS / G > 0 ? BS / G : 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int h = blockIdx.y * kBoundsWaves + wave;
  if (h >= p.hkv) return;
  const int64_t blk = fresh_block(p, blockIdx.z, blockIdx.x);
  if (blk < 0) return;
  const int c = lane % L, g = lane / L;
  const uint16_t* k = static_cast<const uint16_t*>(p.k) + blk * p.ks0 + h * p.ks1 + 8 * c;
  u32x4 x[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k + static_cast<int64_t>(i * G + g) * p.ks2));
  u32x4 lo, hi;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t y[N], l, u;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = x[i][w];
    reduce_bounds<T, L>(y, l, u);
    lo[w] = l;
    hi[w] = u;
  }
  u32x4* dst = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.bounds) + (blk * p.hkv + h) * 2 * D) + c;
  if (g == 0) dst[0] = lo;
  if (g == 1) dst[L] = hi;
}

// The same of a 4-bit pool, four bytes and a scale a lane and token: its values are
// exact in bf16, as which they are compared.
template <typename T, int BS, int D>
__global__ __launch_bounds__(64 * kBoundsWaves) void key_bounds_fp4_kernel(BoundsParams p) {
  constexpr int L = D / 8, G = 64 / L, N = BS / G;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int h = blockIdx.y * kBoundsWaves + wave;
  if (h >= p.hkv) return;
  const int64_t blk = fresh_block(p, blockIdx.z, blockIdx.x);
  if (blk < 0) return;
  const int c = lane % L, g = lane / L;
  const uint8_t* k = static_cast<const uint8_t*>(p.k) + blk * p.ks0 + h * p.ks1;
  uint32_t code[N], byte[N], x[4][N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    code[i] = *reinterpret_cast<const uint32_t*>(k + fp4_key_at<D>(i * G + g, 8 * c));
    byte[i] = k[fp4_key_scale_at<D>(BS, i * G + g, 8 * c)];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float scale = __builtin_bit_cast(float, byte[i] << 23);
    x[0][i] = __builtin_bit_cast(uint32_t, static_cast<bf16x2>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], scale, 0)));
    x[1][i] = __builtin_bit_cast(uint32_t, static_cast<bf16x2>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], scale, 1)));
    x[2][i] = __builtin_bit_cast(uint32_t, static_cast<bf16x2>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], scale, 2)));
    x[3][i] = __builtin_bit_cast(uint32_t, static_cast<bf16x2>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[i], scale, 3)));
  }
  u32x4 lo, hi;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t l, u;
    reduce_bounds<__bf16, L>(x[w], l, u);
    lo[w] = pack2<T>(lo_f32<__bf16>(l), hi_f32<__bf16>(l));
    hi[w] = pack2<T>(lo_f32<__bf16>(u), hi_f32<__bf16>(u));
  }
  u32x4* dst = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.bounds) + (blk * p.hkv + h) * 2 * D) + c;
  if (g == 0) dst[0] = lo;
  if (g == 1) dst[L] = hi;
}

// Any strides: a workgroup a (block, head), a thread a dim.  A token's dims are a load, two
// bytes a thread, so that a whole row takes long (four of 16384 .. 32768 tokens, Hkv 8, D
// 128: token by token off the 16-byte lines 77 us, dim-major, a line a thread, 219; the rows
// kernel 38); what a step completes is bound by the start (64 rows 5.6, 6.0; 3.4).
template <typename T>
__global__ __launch_bounds__(128) void key_bounds_kernel(BoundsParams p) {
  const int h = blockIdx.y, d = threadIdx.x;
  const int64_t blk = fresh_block(p, blockIdx.z, blockIdx.x);
  if (blk < 0) return;
  const uint16_t* k = static_cast<const uint16_t*>(p.k) + blk * p.ks0 + h * p.ks1 + d * p.ks3;
  uint32_t lo = ordered16(k[0]), hi = lo;
  for (int t = 1; t < p.block_size; ++t) {
    const uint32_t x = ordered16(k[t * p.ks2]);
    lo = min16(lo, x);
    hi = max16(hi, x);
  }
  bounds_of<T>(lo, hi);
  uint16_t* dst = static_cast<uint16_t*>(p.bounds) + (blk * p.hkv + h) * 2 * p.head_dim + d;
  dst[0] = static_cast<uint16_t>(lo);
  dst[p.head_dim] = static_cast<uint16_t>(hi);
}

// ============================================================= select ====
struct SelectParams {
  const void* q;
  int64_t qs0, qs1, qs2;
  const void* bounds;  // [block, head, 2, D], contiguous
  const void* bt;
  int64_t bts0, bts1;
  const void* sl;
  int64_t sls;
  int32_t* blocks;  // [request, head, select]
  int32_t* tables;  // the same
  int32_t* lens;    // [request, head]
  uint32_t* keys;   // [request, head, width]
  int sl_i64, hkv, group, block_size, width, select, sinks, recent;
  int64_t num_blocks, block_step;  // block_step: a pool block's distance in KV-head blocks
};

// A row's length and blocks.
struct SelectRow {
  int64_t len;
  int blocks;
};
__device__ __forceinline__ SelectRow select_row(const SelectParams& p, int b) {
  const int64_t cap = static_cast<int64_t>(p.width) * p.block_size;
  int64_t len = load_index_uniform(p.sl, b * p.sls, p.sl_i64);
  len = len < 0 ? 0 : (len < cap ? len : cap);
  return {len, static_cast<int>((len + p.block_size - 1) / p.block_size)};
}

// Scores in an order that whole numbers keep: NaN first, then from the largest down, 0
// behind all of them (-0 counts as 0).
__device__ __forceinline__ uint32_t score_key(double s) {
  const float f = static_cast<float>(s) + 0.f;
  if (f != f) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the L = 8 or 16 neighbouring lanes of a block, in every one of them.
template <int CTRL>
__device__ __forceinline__ double dpp_add_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xf, 0xf, false);
  return x + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
template <int L>
__device__ __forceinline__ double lanes_sum(double x) {
  x = dpp_add_f64<0xb1>(x);   // neighbours
  x = dpp_add_f64<0x4e>(x);   // pairs
  x = dpp_add_f64<0x141>(x);  // quads: lane 7 - i of eight
  if constexpr (L == 16) x = dpp_add_f64<0x140>(x);  // lane 15 - i
  return x;
}

constexpr int kQueryAhead = 4;  // query heads of a thread on their way at once

// Scores of blocks [sinks, last) of one (request, KV head), by WAVES waves of `part` of
// `parts` workgroups: D / 8 lanes a block, eight dims a lane, G = 512 / D blocks a wave at
// once, two of those steps on their way and the ids of a third, behind the query's rows.
// `keep(j, key)` takes them, from one lane a block.  A block is 4 D bytes, and each of its
// 2 D numbers takes a conversion and a multiply-add in 64 bits, which hide behind the
// loads: 16 rows of 16384 .. 32768 tokens, Hkv 8, D 128, blocks of 32, 50 MB in 12.1 us,
// in 32 bits 11.8, without any 11.6.  The bare read would take 7.5; the rest is the start
// (length, ids, bounds in turn, and the queries' sums through LDS).
template <typename T, int D, int WAVES, bool I64, typename Keep>
__device__ __forceinline__ void score_blocks(const SelectParams& p, int b, int h, int last, int part, int parts, Keep keep) {
  constexpr int L = D / 8, G = 64 / L;
  const int lane = threadIdx.x & 63, c = lane % L, g = lane / L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int stride = parts * WAVES * G;
  int j0 = p.sinks + (part * WAVES + wave) * G;
  const T* bounds = static_cast<const T*>(p.bounds) + 8 * c;
  struct Held {
    u32x4 lo, hi;
    bool there;
  };
  auto entry = [&](int j) { return load_block_id<I64>(p.bt, b * p.bts0 + min(j, last - 1) * p.bts1); };
  auto load = [&](Held& x, const BlockId& id) {
    x.there = id.below(p.num_blocks);
    const T* at = bounds + (static_cast<int64_t>(x.there ? id.low : 0) * p.hkv + h) * 2 * D;
    x.lo = *reinterpret_cast<const u32x4*>(at);
    x.hi = *reinterpret_cast<const u32x4*>(at + D);
  };
  Held xa, xb;
  const BlockId ia = entry(j0 + g), ib = entry(j0 + stride + g);
  BlockId ic = entry(j0 + 2 * stride + g);
  load(xa, ia);
  load(xb, ib);
  // Qp and Qm: a thread a dim and every H-th head, then the H parts of each together
  constexpr int H = 64 * WAVES / D;
  __shared__ double s_part[H][2][D], s_sum[2][D];
  {
    const int d = threadIdx.x % D, first = threadIdx.x / D;
    const T* q = static_cast<const T*>(p.q) + b * p.qs0 + static_cast<int64_t>(h * p.group) * p.qs1 + d * p.qs2;
    double u = 0.0, v = 0.0;
    for (int x0 = first; x0 < p.group; x0 += kQueryAhead * H) {
      float y[kQueryAhead];
#pragma unroll
      for (int x = 0; x < kQueryAhead; ++x) {
        const float z = to_f32(q[min(x0 + x * H, p.group - 1) * p.qs1]);
        y[x] = x0 + x * H < p.group ? z : 0.f;
      }
#pragma unroll
      for (int x = 0; x < kQueryAhead; ++x) {  // (a NaN goes into both)
        u += y[x] < 0.f ? 0.f : y[x];
        v += y[x] > 0.f ? 0.f : y[x];
      }
    }
    s_part[first][0][d] = u;
    s_part[first][1][d] = v;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 64 * WAVES) {
      double t = 0.0;
#pragma unroll
      for (int x = 0; x < H; ++x) t += s_part[x][i / D][i % D];
      s_sum[i / D][i % D] = t;
    }
    __syncthreads();
  }
  if (j0 >= last) return;
  double up[8], down[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    up[e] = s_sum[0][8 * c + e];
    down[e] = s_sum[1][8 * c + e];
  }
  auto step = [&](Held& x) -> bool {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fma(up[2 * i], static_cast<double>(lo_f32<T>(x.hi[i])), s);
      s = fma(up[2 * i + 1], static_cast<double>(hi_f32<T>(x.hi[i])), s);
      s = fma(down[2 * i], static_cast<double>(lo_f32<T>(x.lo[i])), s);
      s = fma(down[2 * i + 1], static_cast<double>(hi_f32<T>(x.lo[i])), s);
    }
    const uint32_t key = x.there ? score_key(lanes_sum<L>(s)) : 0u;
    if (c == 0 && j0 + g < last) keep(j0 + g, key);
    load(x, ic);
    ic = entry(j0 + 3 * stride + g);
    j0 += stride;
    return j0 < last;
  };
  while (step(xa) && step(xb)) {
  }
}

constexpr int kScoreWaves = 4;

template <typename T, int D, bool I64>
__global__ __launch_bounds__(64 * kScoreWaves) void block_score_kernel(SelectParams p) {
  const int pair = blockIdx.y, b = pair / p.hkv, h = pair % p.hkv;
  const SelectRow r = select_row(p, b);
  const int last = r.blocks - p.recent;
  if (r.blocks <= p.select || p.sinks + static_cast<int>(blockIdx.x) * kScoreWaves * (512 / D) >= last) return;
  uint32_t* keys = p.keys + static_cast<int64_t>(pair) * p.width;
  score_blocks<T, D, kScoreWaves, I64>(p, b, h, last, blockIdx.x, gridDim.x, [&](int j, uint32_t key) { keys[j] = key; });
}

// A lane's value with the ones below it in the wave, by lane moves: within each 16 lanes,
// then the rows' ends into the rows above (lane 63 has all of them).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x, uint32_t none) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(x), CTRL, ROWS, 0xf, false));
}
template <typename F>
__device__ __forceinline__ uint32_t wave_scan(uint32_t x, uint32_t none, F join) {
  x = join(x, dpp_u32<0x111, 0xf>(x, none));
  x = join(x, dpp_u32<0x112, 0xf>(x, none));
  x = join(x, dpp_u32<0x114, 0xf>(x, none));
  x = join(x, dpp_u32<0x118, 0xf>(x, none));
  x = join(x, dpp_u32<0x142, 0xa>(x, none));
  return join(x, dpp_u32<0x143, 0xc>(x, none));
}

// Exclusive sum over the workgroup, and the whole sum.
template <int THREADS>
__device__ __forceinline__ int pick_scan(int x, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = static_cast<int>(wave_scan(x, 0u, [](uint32_t a, uint32_t b) { return a + b; }));
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int y = s_wave[w];
    before += w < wave ? y : 0;
    total += y;
  }
  __syncthreads();
  return before + upto - x;
}

constexpr int kPickList = 128;  // keys that one wave ranks among each other

// A workgroup a (request, KV head).  The key that the chosen ones reach: a range of keys
// that holds it is cut into at most 2 THREADS equal parts (whole numbers, so that the
// range narrows by as much whatever the scores are), the keys in each counted, and the
// part in which the count from above reaches the number wanted is the next range, until
// it holds so few keys that a wave ranks them directly, or is a single number.  Scores
// spread over the parts, so their counters hardly meet, as they do in the leading bits
// of a radix.  Then the chosen blocks in their order, KEYS THREADS at a time.
// `at_key(j)` is block j's key.
template <int THREADS, int KEYS, bool I64, typename At>
__device__ __forceinline__ void pick_blocks(const SelectParams& p, int pair, const SelectRow& r, At at_key) {
  constexpr int kParts = 2 * THREADS;
  __shared__ int s_count[kParts], s_wave[THREADS / 64], s_part[3];
  __shared__ uint32_t s_list[kPickList], s_least, s_lo[THREADS / 64], s_hi[THREADS / 64];
  const int b = pair / p.hkv, h = pair % p.hkv, tid = threadIdx.x;
  const int lane = tid & 63;
  const bool all = r.blocks <= p.select;
  const int first = p.sinks, last = r.blocks - p.recent;
  uint32_t key[KEYS];  // of the first blocks; later ones are read again
  BlockId id[KEYS];
  auto entry = [&](int j) { return load_block_id<I64>(p.bt, b * p.bts0 + min(j, p.width - 1) * p.bts1); };
#pragma unroll
  for (int i = 0; i < KEYS; ++i) id[i] = entry(KEYS * tid + i);
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = j0 + KEYS * tid + i;
      key[i] = j >= first && j < last ? at_key(j) : 0u;
    }
  };
  constexpr int kSpan = KEYS * THREADS;
  // `take(key)` of every scored block
  auto each = [&](auto take) {
    for (int j0 = 0; j0 < last; j0 += kSpan) {
      if (last > kSpan) load(j0);
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        const int j = j0 + KEYS * tid + i;
        if (j >= first && j < last) take(key[i]);
      }
    }
  };
  uint32_t least = 0;  // the least key chosen, `left` of the `ties` that equal it
  int left = all ? 0 : p.select - p.sinks - p.recent, ties = 0;
  const bool ranks = left > 0;  // (else no block is chosen by its key, and there may be none)
  if (ranks) {
    load(0);
    uint32_t lo = 0xffffffffu, hi = 0;
    each([&](uint32_t k) {
      lo = min(lo, k);
      hi = max(hi, k);
    });
    lo = wave_scan(lo, 0xffffffffu, [](uint32_t a, uint32_t b) { return min(a, b); });
    hi = wave_scan(hi, 0u, [](uint32_t a, uint32_t b) { return max(a, b); });
    if (lane == 63) {
      s_lo[tid >> 6] = lo;
      s_hi[tid >> 6] = hi;
    }
    s_count[2 * tid] = s_count[2 * tid + 1] = 0;
    __syncthreads();
    lo = s_lo[0];
    hi = s_hi[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) {
      lo = min(lo, s_lo[w]);
      hi = max(hi, s_hi[w]);
    }
    constexpr int kPartBits = 31 - __builtin_clz(static_cast<unsigned>(kParts));
    const int bits = 32 - __builtin_clz((hi - lo) | 1u);
    // (four passes at most, each of fewer bits, whatever the keys are)
    for (int shift = max(bits - kPartBits, 0);; shift = max(shift - kPartBits, 0)) {
      each([&](uint32_t k) {
        if (k >= lo && k <= hi) atomicAdd(&s_count[(k - lo) >> shift], 1);
      });
      __syncthreads();
      // thread t: parts kParts - 1 - 2 t and the one below, and how many keys lie above
      const int top = kParts - 1 - 2 * tid;
      const int a = s_count[top], below = s_count[top - 1];
      int total;
      const int above = pick_scan<THREADS>(a + below, s_wave, total);
      s_count[top] = s_count[top - 1] = 0;
      if (above < left && above + a + below >= left) {
        const bool upper = above + a >= left;
        s_part[0] = upper ? top : top - 1;
        s_part[1] = upper ? left - above : left - above - a;
        s_part[2] = upper ? a : below;
      }
      __syncthreads();
      left = s_part[1];
      ties = s_part[2];
      lo += static_cast<uint32_t>(s_part[0]) << shift;
      hi = shift == 0 ? lo : lo + min(hi - lo, (1u << shift) - 1);
      if (shift == 0 || ties <= kPickList) break;
    }
    least = lo;
    if (lo != hi) {  // few keys: each is ranked among them
      __syncthreads();
      if (tid == 0) s_part[2] = 0;
      __syncthreads();
      each([&](uint32_t k) {
        if (k < lo || k > hi) return;
        const int at = atomicAdd(&s_part[2], 1);
        if (at < kPickList) s_list[at] = k;
      });
      __syncthreads();
      for (int i = tid; i < ties; i += THREADS) {
        const uint32_t k = s_list[i];
        int above = 0, same = 0;
        for (int x = 0; x < ties; ++x) {
          above += s_list[x] > k ? 1 : 0;
          same += s_list[x] == k ? 1 : 0;
        }
        if (above < left && above + same >= left) {  // (equal keys write the same)
          s_least = k;
          s_part[0] = left - above;
          s_part[1] = same;
        }
      }
      __syncthreads();
      least = s_least;
      left = s_part[0];
      ties = s_part[1];
    }
  }
  int32_t* blocks = p.blocks + static_cast<int64_t>(pair) * p.select;
  int32_t* tables = p.tables + static_cast<int64_t>(pair) * p.select;
  int n = 0, equal = 0;
  for (int j0 = 0; j0 < r.blocks; j0 += kSpan) {
    if (ranks && r.blocks > kSpan) load(j0);
    const int mine = j0 + KEYS * tid;
    bool chosen[KEYS], tie[KEYS];
    int total, count = 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = mine + i;
      const bool there = j < r.blocks, scored = there && !all && j >= first && j < last;
      tie[i] = ranks && scored && key[i] == least;
      chosen[i] = (there && !scored) || (ranks && scored && key[i] > least) || (tie[i] && left == ties);
      count += chosen[i] ? 1 : 0;
    }
    if (left < ties) {  // the lowest of equal ones
      int same = 0;
#pragma unroll
      for (int i = 0; i < KEYS; ++i) same += tie[i] ? 1 : 0;
      int rank = equal + pick_scan<THREADS>(same, s_wave, total);
      equal += total;
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        if (tie[i]) {
          chosen[i] = rank < left;
          count += chosen[i] ? 1 : 0;
          ++rank;
        }
      }
    }
    int at = n + pick_scan<THREADS>(count, s_wave, total);
    n += total;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      if (chosen[i] && at < p.select) {
        const BlockId x = j0 == 0 ? id[i] : entry(mine + i);
        blocks[at] = mine + i;
        tables[at] = x.below(p.num_blocks) ? static_cast<int32_t>(x.low * p.block_step + h) : -1;
        ++at;
      }
    }
  }
  for (int i = n + tid; i < p.select; i += THREADS) blocks[i] = tables[i] = -1;
  // (the row's last block, which may be partly filled, is always chosen)
  if (tid == 0)
    p.lens[pair] = static_cast<int32_t>(static_cast<int64_t>(n) * p.block_size -
                                        (static_cast<int64_t>(r.blocks) * p.block_size - r.len));
}

template <int THREADS, int KEYS, bool I64>
__global__ __launch_bounds__(THREADS) void block_pick_kernel(SelectParams p) {
  const int pair = blockIdx.x;
  const uint32_t* keys = p.keys + static_cast<int64_t>(pair) * p.width;
  pick_blocks<THREADS, KEYS, I64>(p, pair, select_row(p, pair / p.hkv), [&](int j) { return keys[j]; });
}

// Both in one launch, a workgroup a (request, KV head), the keys in LDS.
template <typename T, int D, int THREADS, int KEYS, bool I64>
__global__ __launch_bounds__(THREADS) void block_select_kernel(SelectParams p) {
  __shared__ uint32_t s_keys[THREADS * KEYS];
  const int pair = blockIdx.x, b = pair / p.hkv, h = pair % p.hkv;
  const SelectRow r = select_row(p, b);
  if (r.blocks > p.select) {
    score_blocks<T, D, THREADS / 64, I64>(p, b, h, r.blocks - p.recent, 0, 1, [&](int j, uint32_t key) { s_keys[j] = key; });
    __syncthreads();
  }
  pick_blocks<THREADS, KEYS, I64>(p, pair, r, [&](int j) { return s_keys[j]; });
}

// ========================================================== host glue ====
namespace {

int check_table(const char* fn, int64_t num_seqs, int64_t num_kv_heads, int64_t width, int64_t block_size,
                int64_t num_blocks, int64_t head_dim, int32_t dtype) {
  if (dtype != FD_DTYPE_F16 && dtype != FD_DTYPE_BF16)
    return set_error(FD_E_UNSUPPORTED, "%s: dtype must be float16 or bfloat16", fn);
  if (head_dim != 64 && head_dim != 128) return set_error(FD_E_UNSUPPORTED, "%s: head_dim must be 64 or 128", fn);
  if (block_size != 8 && block_size != 16 && block_size != 32)
    return set_error(FD_E_UNSUPPORTED, "%s: block_size must be 8, 16 or 32", fn);
  if (num_seqs <= 0 || num_kv_heads <= 0 || width <= 0 || num_blocks <= 0)
    return set_error(FD_E_INVALID, "%s: shapes must be positive", fn);
  if (num_blocks > INT32_MAX) return set_error(FD_E_UNSUPPORTED, "%s: too many blocks", fn);
  if (width > INT32_MAX || width * block_size > INT32_MAX - 4096)
    return set_error(FD_E_UNSUPPORTED, "%s: block tables hold 2^31 tokens or more", fn);
  if (num_seqs > 65535 || num_kv_heads > 65535) return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

int check_select(const fd_block_select_args* args, const char* fn) {
  if (args == nullptr) return set_error(FD_E_INVALID, "%s: args is NULL", fn);
  const fd_block_select_args& a = *args;
  if (a.struct_size != sizeof(fd_block_select_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, a.struct_size,
                     sizeof(fd_block_select_args));
  const int rc = check_table(fn, a.num_seqs, a.num_kv_heads, a.max_blocks_per_seq, a.block_size, a.num_blocks, a.head_dim,
                             a.dtype);
  if (rc != FD_OK) return rc;
  if (a.num_q_heads <= 0 || a.num_q_heads > INT32_MAX || a.num_q_heads % a.num_kv_heads != 0)
    return set_error(FD_E_INVALID, "%s: num_q_heads must be divisible by num_kv_heads", fn);
  if (a.select < 1 || a.sink_blocks < 0 || a.recent_blocks < 1 || a.select > INT32_MAX / 64 ||
      a.sink_blocks > a.select || a.recent_blocks > a.select - a.sink_blocks)
    return set_error(FD_E_INVALID, "%s: select must hold sink_blocks and at least one of recent_blocks", fn);
  if (a.block_step < a.num_kv_heads || a.block_step > INT32_MAX || a.num_blocks * a.block_step > INT32_MAX)
    return set_error(FD_E_UNSUPPORTED, "%s: the KV heads' blocks do not fit 32-bit indices", fn);
  if (!a.q || !a.bounds || !a.block_tables || !a.seq_lens || !a.blocks || !a.tables || !a.lens)
    return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (reinterpret_cast<uintptr_t>(a.bounds) & 15u) return set_error(FD_E_INVALID, "%s: bounds must be 16-byte aligned", fn);
  if (a.num_seqs * a.num_kv_heads > 65535) return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

// Whether a block can be chosen by its score: else every row has all of its blocks, or
// its sinks and recent ones, and no key is made or read.
bool any_scored(const fd_block_select_args& a) {
  return a.max_blocks_per_seq > a.select && a.select > a.sink_blocks + a.recent_blocks;
}

// Both in one launch for short tables: a launch less, and a CU has few blocks to score.
// MI355X, us of two launches / one: 2 pairs of 128 blocks 7.3 / 7.3, of 256 7.4 / 8.9 (and
// 2 less on the host), of 512 7.5 / 11.9; 64 of 256 9.1 / 9.1, of 512 9.9 / 12.2; 200 of 128
// 10.0 / 7.7; 256 of 512 18.9 / 16.7; 512 of 256 19.1 / 16.1; 128 of 1024 16.8 / 19.3.
bool select_whole(const fd_block_select_args& a) {
  const int64_t width = a.max_blocks_per_seq;
  return any_scored(a) && (width <= 256 || (width <= 512 && a.num_seqs * a.num_kv_heads >= device_cus()));
}

// (a table no wider than the list: every row has all of its blocks, and no keys)
int64_t select_words(const fd_block_select_args& a) {
  return a.max_blocks_per_seq > a.select ? a.num_seqs * a.num_kv_heads * a.max_blocks_per_seq : 0;
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_key_bounds(const fd_key_bounds_args* args, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_key_bounds";
  if (args == nullptr) return set_error(FD_E_INVALID, "%s: args is NULL", fn);
  const fd_key_bounds_args& a = *args;
  if (a.struct_size != sizeof(fd_key_bounds_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, a.struct_size,
                     sizeof(fd_key_bounds_args));
  const int rc = check_table(fn, a.num_seqs, a.num_kv_heads, a.max_blocks_per_seq, a.block_size, a.num_blocks, a.head_dim,
                             a.dtype);
  if (rc != FD_OK) return rc;
  if (a.new_tokens < 0) return set_error(FD_E_INVALID, "%s: new_tokens must be non-negative", fn);
  if (a.fp4 != 0 && a.fp4 != 1) return set_error(FD_E_INVALID, "%s: fp4 must be 0 or 1", fn);
  if (!a.k_cache || !a.block_tables || !a.seq_lens || !a.bounds) return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (reinterpret_cast<uintptr_t>(a.bounds) & 15u) return set_error(FD_E_INVALID, "%s: bounds must be 16-byte aligned", fn);
  if (a.fp4) {
    const int rc = check_fp4_caches(fn, a.head_dim, a.block_size, a.num_blocks, a.num_kv_heads, a.k_cache, a.k_stride,
                                    a.k_cache, a.k_stride);
    if (rc != FD_OK) return rc;
  }
  // blocks that the new tokens of a row may complete
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  const int64_t fresh = a.new_tokens < cap ? a.new_tokens : cap;
  const int64_t touched = (fresh + a.block_size - 1) / a.block_size;
  if (touched == 0) return FD_OK;
  if (!grid_fits(touched, 64 * kBoundsWaves)) return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  BoundsParams p{};
  p.k = a.k_cache;
  p.ks0 = a.k_stride[0];
  p.ks1 = a.k_stride[1];
  p.ks2 = a.k_stride[2];
  p.ks3 = a.k_stride[3];
  p.bt = a.block_tables;
  p.bts0 = a.block_tables_stride[0];
  p.bts1 = a.block_tables_stride[1];
  p.sl = a.seq_lens;
  p.sls = a.seq_lens_stride;
  p.bounds = a.bounds;
  p.bt_i64 = a.block_tables_dtype == FD_INDEX_I64;
  p.sl_i64 = a.seq_lens_dtype == FD_INDEX_I64;
  p.hkv = static_cast<int>(a.num_kv_heads);
  p.head_dim = static_cast<int>(a.head_dim);
  p.block_size = static_cast<int>(a.block_size);
  p.width = static_cast<int>(a.max_blocks_per_seq);
  p.num_blocks = a.num_blocks;
  p.new_tokens = fresh;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const bool rows = a.fp4 || (a.k_stride[3] == 1 && a.k_stride[0] % 8 == 0 && a.k_stride[1] % 8 == 0 &&
                              a.k_stride[2] % 8 == 0 && (reinterpret_cast<uintptr_t>(a.k_cache) & 15u) == 0);
  const int64_t heads = rows ? (a.num_kv_heads + kBoundsWaves - 1) / kBoundsWaves : a.num_kv_heads;
  const dim3 grid(static_cast<unsigned>(touched), static_cast<unsigned>(heads), static_cast<unsigned>(a.num_seqs));
  auto launch = [&](auto type) {
    using T = decltype(type);
    auto go = [&](auto kernel, int threads) { dispatch(kernel, grid, dim3(threads), stream, nullptr, nullptr, p); };
    auto sized = [&](auto block) {
      constexpr int BS = decltype(block)::value, kThreads = 64 * kBoundsWaves;
      if (a.fp4)
        a.head_dim == 64 ? go(key_bounds_fp4_kernel<T, BS, 64>, kThreads) : go(key_bounds_fp4_kernel<T, BS, 128>, kThreads);
      else
        a.head_dim == 64 ? go(key_bounds_rows_kernel<T, BS, 64>, kThreads) : go(key_bounds_rows_kernel<T, BS, 128>, kThreads);
    };
    if (!rows)
      go(key_bounds_kernel<T>, static_cast<int>(a.head_dim));
    else if (a.block_size == 8)
      sized(std::integral_constant<int, 8>{});
    else if (a.block_size == 16)
      sized(std::integral_constant<int, 16>{});
    else
      sized(std::integral_constant<int, 32>{});
  };
  a.dtype == FD_DTYPE_BF16 ? launch(__bf16{}) : launch(_Float16{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return FD_OK;
}

extern "C" int fd_block_select_words(const fd_block_select_args* args, int64_t* words) {
  static const char* fn = "fd_block_select_words";
  const int rc = check_select(args, fn);
  if (rc != FD_OK) return rc;
  if (words == nullptr) return set_error(FD_E_INVALID, "%s: words is NULL", fn);
  *words = select_words(*args);
  return FD_OK;
}

extern "C" int fd_block_select(const fd_block_select_args* args, int32_t* workspace, int64_t words, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_block_select";
  const int rc = check_select(args, fn);
  if (rc != FD_OK) return rc;
  const fd_block_select_args& a = *args;
  if (select_words(a) > 0 &&
      (workspace == nullptr || words < select_words(a) || (reinterpret_cast<uintptr_t>(workspace) & 3u)))
    return set_error(FD_E_INVALID, "%s: needs a workspace of %lld words", fn, static_cast<long long>(select_words(a)));
  SelectParams p{};
  p.q = a.q;
  p.qs0 = a.q_stride[0];
  p.qs1 = a.q_stride[1];
  p.qs2 = a.q_stride[2];
  p.bounds = a.bounds;
  p.bt = a.block_tables;
  p.bts0 = a.block_tables_stride[0];
  p.bts1 = a.block_tables_stride[1];
  p.sl = a.seq_lens;
  p.sls = a.seq_lens_stride;
  p.blocks = a.blocks;
  p.tables = a.tables;
  p.lens = a.lens;
  p.keys = reinterpret_cast<uint32_t*>(workspace);
  p.sl_i64 = a.seq_lens_dtype == FD_INDEX_I64;
  p.hkv = static_cast<int>(a.num_kv_heads);
  p.group = static_cast<int>(a.num_q_heads / a.num_kv_heads);
  p.block_size = static_cast<int>(a.block_size);
  p.width = static_cast<int>(a.max_blocks_per_seq);
  p.select = static_cast<int>(a.select);
  p.sinks = static_cast<int>(a.sink_blocks);
  p.recent = static_cast<int>(a.recent_blocks);
  p.num_blocks = a.num_blocks;
  p.block_step = a.block_step;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int64_t pairs = a.num_seqs * a.num_kv_heads;
  const bool bf = a.dtype == FD_DTYPE_BF16;
  const dim3 grid(static_cast<unsigned>(pairs));
  auto by_index = [&](auto launch) {  // kernels by the block ids' type
    a.block_tables_dtype == FD_INDEX_I64 ? launch(std::true_type{}) : launch(std::false_type{});
  };
  if (select_whole(a)) {
    auto go = [&](auto kernel) { dispatch(kernel, grid, dim3(512), stream, nullptr, nullptr, p); };
    by_index([&](auto index) {
      constexpr bool I64 = decltype(index)::value;
      if (a.head_dim == 64)
        bf ? go(block_select_kernel<__bf16, 64, 512, 1, I64>) : go(block_select_kernel<_Float16, 64, 512, 1, I64>);
      else
        bf ? go(block_select_kernel<__bf16, 128, 512, 1, I64>) : go(block_select_kernel<_Float16, 128, 512, 1, I64>);
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return FD_OK;
  }
  if (any_scored(a)) {
    // at most four workgroups a CU
    const int64_t step = kScoreWaves * (512 / a.head_dim);
    const int64_t most = (a.max_blocks_per_seq + step - 1) / step;
    int64_t parts = (4 * device_cus() + pairs - 1) / pairs;
    parts = parts < most ? parts : most;
    const dim3 shares(static_cast<unsigned>(parts), static_cast<unsigned>(pairs));
    auto score = [&](auto kernel) { dispatch(kernel, shares, dim3(64 * kScoreWaves), stream, nullptr, nullptr, p); };
    by_index([&](auto index) {
      constexpr bool I64 = decltype(index)::value;
      if (a.head_dim == 64)
        bf ? score(block_score_kernel<__bf16, 64, I64>) : score(block_score_kernel<_Float16, 64, I64>);
      else
        bf ? score(block_score_kernel<__bf16, 128, I64>) : score(block_score_kernel<_Float16, 128, I64>);
    });
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  }
  // Threads for a full table row's blocks, one to four neighbours each (a thread's keys are
  // counted one after the other).  MI355X, both launches, us with 256 x 4, 512 x 2, 512 x 8,
  // 1024 x 1, 1024 x 4 threads x keys: 2 pairs of 256 blocks 7.8, 7.7, 9.7, 8.6, 9.8; 64 of
  // 1024 14.5, 12.8, 15.1, 13.6, 14.6; 512 of 256 19.3, 19.5, 22.1, 23.4, 25.7; 2 of 4096
  // 17.0, 13.4, 12.9, 13.6, 11.1; 32 of 4096 28.7, 24.6, 23.5, 24.3, 21.8.
  auto pick = [&](auto kernel, int threads) { dispatch(kernel, grid, dim3(threads), stream, nullptr, nullptr, p); };
  const int64_t width = a.max_blocks_per_seq;
  by_index([&](auto index) {
    constexpr bool I64 = decltype(index)::value;
    if (width <= 512)
      pick(block_pick_kernel<512, 1, I64>, 512);
    else if (width <= 1024)
      pick(block_pick_kernel<512, 2, I64>, 512);
    else if (width <= 2048)
      pick(block_pick_kernel<1024, 2, I64>, 1024);
    else
      pick(block_pick_kernel<1024, 4, I64>, 1024);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return FD_OK;
}
