// Single-token decode attention over a 4-bit cache (fp4_format.h), for gfx950.
//
// With s = scale * q.k, x = s log2(e), a row's tokens are cut into chunks of 32-token
// tiles, one a workgroup; each leaves a reference M at or above its max x, L = sum
// 2^(x - M) and sum 2^(x - M) v, and a second launch joins them (join_rows): out =
// sum_c 2^(M_c - M) acc_c / sum_c 2^(M_c - M) L_c.  Calls of one chunk a row store it at once.  Chunks are cut by the
// table's width, or by the rows' lengths (Fp4Item).
#include <algorithm>

#include "decode_host.h"
#include "fp4_format.h"

namespace fd {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp4Args {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  void* out;
  float* acc;
  float2* stats;
  int64_t qs0, qs1, qs2, ks0, ks1, vs0, vs1, os0, os1, os2;  // ks, vs: bytes
  int32_t q_rows, out_rows;  // rows of unit stride on 16-byte lines
  int32_t hq, group, head_blocks, num_blocks, width, cap;
  int32_t wide;  // the bits of a block id's high word: -1 of 64-bit ids, else 0
  // items > 0: chunks by the rows' lengths (Fp4Item)
  int32_t rows, items, per_cu, floor, least;
  int32_t* live;               // 32 times each row's chunks, for the join
  // sm_scale log2(e) as a sign, which goes into the query (0 makes that zero), and a
  // positive factor, under which the largest product is the largest score
  float sign, scale_log2;
};

constexpr int kFp4Waves = 4;
constexpr int kFp4ItemRows = 256;  // of calls with items, at most

// ------------------------------------------------------------- queries --
// A query is kept as a sum of 8-bit floating-point terms, so that q.k runs on the
// scaled matrix instruction with the cache's bytes as they lie in memory.  A group of
// 32 dims whose largest magnitude lies in [2^E, 2^(E+1)) is scaled by 2^(7-E); its
// first term has 4 significant bits, what is left is at most 2^-5 of that range and is
// scaled up by as much for the next.  Two terms hold a bf16 value exactly, three an
// fp16 one, down to 2^-22 of the group's largest.
//
// The instruction's 8-bit operand of lane (c, h) (column c = query head): k = 16 h + i
// in its first half, 64 + 16 h + i in its second; the scale of k's 32-block g comes
// from lane (c, g).  128-dim heads: k = dim, one product a term.  64-dim heads: k =
// dim in the first 64, and again in the second, for the next term; the keys enter
// twice.
template <typename T, int D>
struct Fp4Query {
  static constexpr int kTerms = sizeof(T) == 2 && std::is_same_v<T, __bf16> ? 2 : 3;
  static constexpr int kProducts = D == 128 ? kTerms : (kTerms + 1) / 2;
  i32x8 code[kProducts];
  int scale[kProducts];
};

// A lane's dims of a query row, as loaded: 16 at 16 h, and of 128-dim heads 16 at 64 + 16 h.
template <int D>
struct Fp4QueryRow {
  u32x4 w[D / 32];
};

template <typename T, int D>
__device__ __forceinline__ Fp4QueryRow<D> fp4_query_load(const T* row, int64_t step, bool rows, int h) {
  Fp4QueryRow<D> q;
  const int d0 = 16 * h;
  if (rows) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q.w[i] = *reinterpret_cast<const u32x4*>(row + d0 + 64 * (i >> 1) + 8 * (i & 1));
  } else {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T* at = row + (d0 + 64 * (i >> 1) + 8 * (i & 1) + 2 * j) * step;
        q.w[i][j] = __builtin_bit_cast(uint16_t, at[0]) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, at[step])) << 16;
      }
  }
  return q;
}

template <typename T>
__device__ __forceinline__ void fp4_query_piece(const u32x4& a, const u32x4& b, float (&x)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = lo_f32<T>(a[j]);
    x[2 * j + 1] = hi_f32<T>(a[j]);
    x[8 + 2 * j] = lo_f32<T>(b[j]);
    x[9 + 2 * j] = hi_f32<T>(b[j]);
  }
}

// Splits 16 values of a group (whose other 16 are in lane ^ 16), times `sign` (1, -1 or
// 0), into terms of four words and returns the first term's scale byte.
template <int TERMS>
__device__ __forceinline__ int fp4_query_split(float (&x)[16], float sign, uint32_t (&word)[TERMS][4]) {
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) amax = max(amax, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
  amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16, 64)));
  const bool odd = amax >= 0x7f800000u;  // a NaN or an infinity: every score is NaN
  // (down to what leaves the last term's scale a byte; bf16 values, whose steps end at
  // 2^-133, stay exact below it, fp16 ones end at 2^-24)
  const int e = max(static_cast<int>(amax >> 23) - 127, 5 * (TERMS - 1) - 120);
  const float unit = sign * __builtin_bit_cast(float, static_cast<uint32_t>(7 - e + 127) << 23);
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = odd ? 0.f : x[j] * unit;
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      int code = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w], x[4 * w + 1], 0, false);
      code = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2], x[4 * w + 3], code, true);
      word[t][w] = static_cast<uint32_t>(code);
      const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(code, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(code, true);
      x[4 * w] = (x[4 * w] - a[0]) * 32.f;
      x[4 * w + 1] = (x[4 * w + 1] - a[1]) * 32.f;
      x[4 * w + 2] = (x[4 * w + 2] - b[0]) * 32.f;
      x[4 * w + 3] = (x[4 * w + 3] - b[1]) * 32.f;
    }
  }
  return odd ? 0xff : e + 120;
}

// (a NaN's scale byte stays 255; a fourth term, which fp16 calls of 64-dim heads pad theirs
// with, is zeros)
__device__ __forceinline__ int fp4_term_scale(int first, int term) { return first == 0xff ? first : max(first - 5 * term, 0); }

template <typename T, int D>
__device__ __forceinline__ Fp4Query<T, D> fp4_query(const Fp4QueryRow<D>& row, float sign, int lane) {
  constexpr int N = Fp4Query<T, D>::kTerms;
  const int h = lane >> 4, c = lane & 15;
  Fp4Query<T, D> q;
  float x[16];
  uint32_t lo[N][4];
  fp4_query_piece<T>(row.w[0], row.w[1], x);
  const int s_lo = fp4_query_split<N>(x, sign, lo);  // of dims [32 (h / 2), + 32)
  if constexpr (D == 128) {
    uint32_t hi[N][4];
    fp4_query_piece<T>(row.w[2], row.w[3], x);
    const int s_hi = fp4_query_split<N>(x, sign, hi);  // of dims [64 + 32 (h / 2), + 32)
    const int src = c + 32 * (h & 1);
    const int a = __shfl(s_lo, src, 64), b = __shfl(s_hi, src, 64);
    const int mine = h < 2 ? a : b;
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        q.code[t][w] = static_cast<int>(lo[t][w]);
        q.code[t][4 + w] = static_cast<int>(hi[t][w]);
      }
      q.scale[t] = fp4_term_scale(mine, t);
    }
  } else {
    const int mine = __shfl(s_lo, c + 32 * (h & 1), 64);
#pragma unroll
    for (int t = 0; t < (N + 1) / 2; ++t) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        q.code[t][w] = static_cast<int>(lo[2 * t][w]);
        q.code[t][4 + w] = 2 * t + 1 < N ? static_cast<int>(lo[min(2 * t + 1, N - 1)][w]) : 0;
      }
      q.scale[t] = fp4_term_scale(mine, 2 * t + (h >> 1));
    }
  }
  return q;
}

// --------------------------------------------------------------- units --
// A unit is 32 tokens, two tiles of 16.  Lane (c, g): of tile m, key token c, dims
// [32 g, + 32) (64-dim heads: g % 2), one byte of scale; values of tokens 4 g .. 4 g + 3,
// dims [(D / 16) c, + D / 16), and their four scale bytes as a word.
template <int D>
struct Fp4Unit {
  using Values = std::conditional_t<D == 128, u32x4, u32x2>;
  u32x4 k[2];
  uint32_t ks[2];
  Values v[2];
  uint32_t vs[2];
  uint32_t there;  // bit m: this lane's tokens of tile m lie in a block of the pool
  bool all;        // the whole unit does
};

// Block ids of a unit, -1 past the chunk.
template <int BS>
struct Fp4Pages {
  BlockId id[32 / BS];
};

template <int BS>
__device__ __forceinline__ Fp4Pages<BS> fp4_pages(const void* bt, int64_t row, int64_t step, int i64, int width, int tok0,
                                                  bool live) {
  Fp4Pages<BS> p;
#pragma unroll
  for (int i = 0; i < 32 / BS; ++i)
    p.id[i] = live ? load_block_id_uniform(bt, row + static_cast<int64_t>(min(tok0 / BS + i, width - 1)) * step, i64)
                   : BlockId{-1, -1};
  return p;
}

// A descriptor of a block's bytes from a uniform address; empty (reads give zeros) where
// `there` is 0, else -1.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t fp4_rsrc(const uint8_t* at, int there) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at), 0, there, 0x00020000);
}
template <bool NT, typename V>
__device__ __forceinline__ V fp4_load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at, uint32_t from) {
  if constexpr (sizeof(V) == 16)
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, from, NT ? 2 : 0));
  else
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, from, NT ? 2 : 0));
}

// Blocks of 16 and 32 tokens hold a tile: a descriptor of the block and the lane's offset
// in it, which is the same for every unit (with an address computed for each unit the
// registers that hold it tie its loads to the unit before).  Of blocks of 8 the lane's
// half of the tile picks one; those outside the pool read block 0.
template <int BS, int D, bool NT>
__device__ __forceinline__ void fp4_load_unit(const Fp4Args& a, const uint8_t* kh, const uint8_t* vh, const Fp4Pages<BS>& p,
                                              int c, int g, Fp4Unit<D>& t) {
  using Values = typename Fp4Unit<D>::Values;
  constexpr int kKeyScales = BS * D / 2, kValueScales = BS * D / 2;
  const int kg = D == 128 ? g : g & 1, vg = (D / 16) * c / 32;
  t.there = 0;
  t.all = true;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if constexpr (BS >= 16) {
      const int32_t id = p.id[BS == 32 ? 0 : m].low, far = p.id[BS == 32 ? 0 : m].high & a.wide;
      // -1 for a block of the pool, else 0, by whole-number arithmetic (opaque in the middle:
      // a comparison's result is selected in a vector register, and the descriptor with it)
      int past = id - a.num_blocks;
      asm("" : "+s"(past));
      const int ok = (past & ~id & ~(far | -far)) >> 31;
      const int64_t blk = id & ok;
      const int tile = BS == 32 ? m : 0;  // of the block
      const __amdgpu_buffer_rsrc_t kr = fp4_rsrc(kh + blk * a.ks0, ok), vr = fp4_rsrc(vh + blk * a.vs0, ok);
      t.k[m] = fp4_load<NT, u32x4>(kr, c * (D / 2) + 16 * kg, tile * 8 * D);
      t.ks[m] = __builtin_amdgcn_raw_buffer_load_b8(kr, c * (D / 32) + kg, kKeyScales + tile * (D / 2), 0);
      t.v[m] = fp4_load<NT, Values>(vr, g * (2 * D) + c * (D / 8), tile * 8 * D);
      t.vs[m] = __builtin_amdgcn_raw_buffer_load_b32(vr, g * (D / 8) + 4 * vg, kValueScales + tile * (D / 2), 0);
      t.there |= static_cast<uint32_t>(ok) & (1u << m);
      t.all = t.all && ok;
    } else {
      const int32_t i0 = p.id[2 * m].low, i1 = p.id[2 * m + 1].low;
      const bool ok0 = i0 >= 0 && i0 < a.num_blocks && (p.id[2 * m].high & a.wide) == 0;
      const bool ok1 = i1 >= 0 && i1 < a.num_blocks && (p.id[2 * m + 1].high & a.wide) == 0;
      const int64_t b0 = ok0 ? i0 : 0, b1 = ok1 ? i1 : 0;
      const uint8_t* kp = kh + (c < 8 ? b0 : b1) * a.ks0;
      const uint8_t* vp = vh + (g < 2 ? b0 : b1) * a.vs0;
      t.k[m] = kv_load<NT, u32x4>(kp + (c & 7) * (D / 2) + 16 * kg);
      t.ks[m] = kp[kKeyScales + (c & 7) * (D / 32) + kg];
      t.v[m] = kv_load<NT, Values>(vp + (g & 1) * (2 * D) + c * (D / 8));
      t.vs[m] = *reinterpret_cast<const uint32_t*>(vp + kValueScales + (g & 1) * (D / 8) + 4 * vg);
      t.there |= (g < 2 ? ok0 : ok1) ? 1u << m : 0u;
      t.all = t.all && ok0 && ok1;
    }
  }
}

// Dims [2 w, 2 w + 1] of a lane's value piece of token i, as bf16 (exact).
template <int D>
__device__ __forceinline__ uint32_t fp4_value_pair(const typename Fp4Unit<D>::Values& v, int i, int w, float scale) {
  const uint32_t word = D == 128 ? v[i] : v[i >> 1];
  const int at = D == 128 ? w : 2 * (i & 1) + w;
  switch (at) {  // (the byte is an immediate)
    case 0: return __builtin_bit_cast(uint32_t, static_cast<bf16x2_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0)));
    case 1: return __builtin_bit_cast(uint32_t, static_cast<bf16x2_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1)));
    case 2: return __builtin_bit_cast(uint32_t, static_cast<bf16x2_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2)));
    default: return __builtin_bit_cast(uint32_t, static_cast<bf16x2_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3)));
  }
}

// Online softmax of a unit's scores.  st.m is a reference that no score passes, not the
// maximum: where one does, it moves to kRescaleSlack above the new maximum, so that it
// moves, and the accumulator is scaled, in few units (a wave moves for any of its 16
// heads: moving it with every new maximum costs 64 rows of 8192 tokens, Hq 32, Hkv 8,
// 95 us instead of 87), and no probability is above 1 (one of 2^8 would carry values of
// 2^120 past the largest number).
// Scores are rounded before the reference goes off: in one multiply-add the largest one's
// would be off by the rounding of a product that it was not, half a step of it, which is
// more than an exponent where scores pass 2^31.
template <int D>
__device__ __forceinline__ void fp4_softmax(const float (&sc)[8], float scale_log2, float (&pr)[8], WaveState<D>& st) {
#pragma clang fp contract(off)
  float x[8], mx;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = sc[i] * scale_log2;
    mx = i == 0 ? x[0] : fmaxf(mx, x[i]);
  }
  mx = column_max(mx);
  const bool move = mx > st.m;
  if (__ballot(move)) {
    const float to = move ? mx + kRescaleSlack : st.m;
    // (while st.m is -inf, acc and l are zero)
    const float alpha = st.m == -INFINITY ? 0.f : exp2_fast(st.m - to);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) st.acc[n] *= alpha;
    st.l *= alpha;
    st.m = to;
  }
  const float m_use = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    pr[i] = exp2_fast(x[i] - m_use);
    st.l += pr[i];
  }
}

// Two numbers rounded to bf16, as a word (pack2 of bf16 in one instruction).
__device__ __forceinline__ uint32_t fp4_pack(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, bf16x2_t));
}

template <typename T, int D>
__device__ __forceinline__ void fp4_process(Fp4Unit<D>& t, const Fp4Query<T, D>& q, float scale_log2, int tok0, int last,
                                            int g, WaveState<D>& st) {
  float sc[8], pr[8];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    i32x8 key = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) key[w] = static_cast<int>(t.k[m][w]);
    // formats: 4 is e2m1 (the keys), 0 is e4m3 (the query's terms)
#pragma unroll
    for (int n = 0; n < Fp4Query<T, D>::kProducts; ++n)
      s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(key, q.code[n], s, 4, 0, 0, static_cast<int>(t.ks[m]), 0,
                                                           q.scale[n]);
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[4 * m + i] = s[i];
  }
  // tokens past the end or in no block: no score, and a scale that is a number (their
  // bytes may say NaN, and 0 * NaN is NaN)
  if (!t.all || tok0 + 31 > last) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint32_t keep = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool live = (t.there >> m & 1u) && tok0 + 16 * m + 4 * g + i <= last;
        sc[4 * m + i] = live ? sc[4 * m + i] : -INFINITY;
        keep |= live ? 0xffu << (8 * i) : 0u;
      }
      t.vs[m] &= keep;
    }
  }
  fp4_softmax<D>(sc, scale_log2, pr, st);
  u32x4 p;
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = fp4_pack(pr[2 * j], pr[2 * j + 1]);
  // the values' levels are exact in bf16 over all of its range, which fp16 is too small
  // for; what the probabilities lose to it enters as a second term (one term: 64 rows of
  // 8192 tokens, Hq 32, Hkv 8, bf16 87 us for 88, 64-dim heads 52 for 55, and an error of
  // 0.0023 for 0.0017, which is that of the result's own rounding)
  u32x4 rest;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    rest[j] = fp4_pack(pr[2 * j] - lo_f32<__bf16>(p[j]), pr[2 * j + 1] - hi_f32<__bf16>(p[j]));
  // (the conversion goes by its scale's exponent bits alone: the byte moves there, and
  // what lies in the others does not matter)
  float scale[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    scale[i] = __builtin_bit_cast(float, __builtin_amdgcn_alignbit(t.vs[i >> 2], t.vs[i >> 2], (8 * (i & 3) + 9) & 31));
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fp4_value_pair<D>(t.v[i >> 2], i & 3, w, scale[i]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t sel = e ? 0x07060302u : 0x05040100u;
      u32x4 vt;
#pragma unroll
      for (int j = 0; j < 4; ++j) vt[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], sel);
      st.acc[2 * w + e] = mfma16x16x32<__bf16>(vt, p, st.acc[2 * w + e]);
      st.acc[2 * w + e] = mfma16x16x32<__bf16>(vt, rest, st.acc[2 * w + e]);
    }
  }
}

// ---------------------------------------------------------------- items --
// Chunks by the rows' lengths: every row is cut after each `per` of its tiles, and item i
// is the i-th of all rows' chunks, of which there are at most a.items.  Each workgroup
// finds its own from the lengths alone, with whole numbers, so that all find the same.  `per` is what a CU has to read in all over a.per_cu, but at
// least a.floor tiles, or where a CU has less than that, all of it; and never less than
// a.least, so that the rows' partials have a bounded place.
struct Fp4Item {
  int row, len, chunk, per;
};

// Inclusive sums over the lanes of a wave: in rows of 16, then over those.
__device__ __forceinline__ int fp4_sums(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // one lane on
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // two
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // four
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // eight
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lanes 15, 47 to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
  return x;
}

// Of R rows a lane, neighbours: at most 64 R.
template <int R>
__device__ __forceinline__ Fp4Item fp4_item(const void* sl, int32_t sls, int sl_i64, const Fp4Args& a, int item, int lane,
                                            bool writes) {
  int len[R], tiles[R], mine[R], sum = 0, full = 0;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int row = R * lane + k;
    len[k] = 0;
    // (a 64-bit length's low half, as everywhere)
    if (row < a.rows) len[k] = load_index(sl, static_cast<int64_t>(row) * sls, sl_i64);
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
    len[k] = len[k] < 0 ? 0 : (len[k] < a.cap ? len[k] : a.cap);
    tiles[k] = (len[k] + 31) >> 5;
    sum += tiles[k];
    full += __builtin_popcountll(__ballot(tiles[k] > 0));
  }
  sum = __builtin_amdgcn_readlane(fp4_sums(sum), 63);
  const int share = (sum + a.items - 1) / a.items;
  int per = max(share >= a.floor ? share : min(a.floor, a.per_cu * share), a.least), own, ends;
  // a row's last chunk is half full on average, so that the share may not do, nor one
  // that allows for that; one that allows for a chunk more of every row does (a.items
  // is more than the rows)
  for (int t = 0;; ++t) {
    own = 0;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      mine[k] = static_cast<int>(static_cast<uint32_t>(tiles[k] + per - 1) / static_cast<uint32_t>(per));
      own += mine[k];
    }
    ends = fp4_sums(own);
    if (t == 2 || __builtin_amdgcn_readlane(ends, 63) <= a.items) break;
    per = max(per, sum / (a.items - (t == 0 ? full / 2 : full)) + 1);
  }
  const int begins = ends - own;
  if (writes) {
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (R * lane + k < a.rows) a.live[R * lane + k] = 32 * mine[k];
  }
  // the last lane that begins at or before the item (one without chunks begins where the
  // next one does; lane 0 begins at 0), and its rows in turn
  const int holder = 63 - __builtin_clzll(__ballot(begins <= item));
  const bool there = item < __builtin_amdgcn_readlane(ends, 63);
  Fp4Item r;
  r.row = R * holder;
  r.len = __builtin_amdgcn_readlane(len[0], holder);
  r.chunk = item - __builtin_amdgcn_readlane(begins, holder);
  r.per = per;
  bool on = true;
#pragma unroll
  for (int k = 0; k + 1 < R; ++k) {
    const int before = __builtin_amdgcn_readlane(mine[k], holder);
    on = on && r.chunk >= before;
    r.chunk -= on ? before : 0;
    r.row += on ? 1 : 0;
    r.len = on ? __builtin_amdgcn_readlane(len[k + 1], holder) : r.len;
  }
  // an item behind all takes a row's first chunk, without tokens (its own would start
  // behind any table)
  r.row = min(r.row, a.rows - 1);
  r.len = there ? r.len : 0;
  r.chunk = there ? r.chunk : 0;
  return r;
}

// One workgroup of four waves per (request, KV head, 16 query heads, chunk), its waves
// taking units in turn, the next one's bytes on their way.  Large calls are bound by HBM
// reads: 64 rows of 8192 tokens, Hq 32, Hkv 8, D 128, 570 MB in 88 us, 6.5 TB/s, with the
// vector units half busy (64 of a unit's 167 vector instructions turn values into bf16
// operands; keys take none, a lane's 16 bytes and scale are the product's operand); two
// units ahead are no faster, cached loads slower (103 us).  Small ones by their start
// (lengths and block ids, K/V, 4 us) and the join (3 us); groups of up to 16 heads cost
// what one head does, and larger ones read K and V again for every 16 (16 rows of 8192
// tokens, Hkv 1, 64-dim fp16: 16 heads 9.4 us, 32 12.1, 71 18.1; cached loads the same).
template <typename T, int BS, int D, bool NT>
__global__ __launch_bounds__(64 * kFp4Waves, 3) void fp4_decode_kernel(const void* sl, const void* bt, int64_t bts0, int64_t bts1,
                                                                    int32_t sls, int32_t i64, int32_t chunks,
                                                                    int32_t chunk_tiles, Fp4Args a) {
  constexpr int P = acc_pitch<D>(), W = kFp4Waves;
  __shared__ __attribute__((aligned(16))) float s_acc[W * 16 * P];
  __shared__ float s_m[W][16], s_l[W][16];
  int b = blockIdx.z, chunk = blockIdx.x / a.head_blocks;
  const int kvh = blockIdx.y, hb = blockIdx.x - chunk * a.head_blocks;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int head0 = 16 * hb;
  // columns past the group's last head take its first; their results are dropped
  const int head = head0 + c < a.group ? head0 + c : 0;
  // the length and the first block ids together, then the query and the first unit, and
  // the query is split while that is on its way
  int len;
  if (a.items > 0) {
    const bool first = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && wave == 0;
    const Fp4Item item = a.rows <= 64 ? fp4_item<1>(sl, sls, i64 & 1, a, blockIdx.z, lane, first)
                                      : fp4_item<kFp4ItemRows / 64>(sl, sls, i64 & 1, a, blockIdx.z, lane, first);
    b = item.row;
    len = item.len;
    chunk = item.chunk;
    chunk_tiles = item.per;
  } else {
    len = load_index_uniform(sl, static_cast<int64_t>(b) * sls, i64 & 1);
  }
  const int64_t table_row = b * bts0;
  int u = chunk * chunk_tiles + wave;
  // (a chunk behind the table's last tile takes that one's: its tokens may pass 2^31)
  Fp4Pages<BS> pages = fp4_pages<BS>(bt, table_row, bts1, i64 >> 1, a.width, 32 * min(u, (a.cap - 1) >> 5), true);
  const T* row = static_cast<const T*>(a.q) + b * a.qs0 + (static_cast<int64_t>(kvh) * a.group + head) * a.qs1;
  const Fp4QueryRow<D> query = fp4_query_load<T, D>(row, a.qs2, a.q_rows, g);
  len = len < 0 ? 0 : (len < a.cap ? len : a.cap);
  const int tiles = (len + 31) >> 5;
  const int begin = chunk * chunk_tiles, end = min(begin + chunk_tiles, tiles);
  if (begin >= end && chunks > 1) return;  // the join reads a row's own chunks only
  const uint8_t* kh = a.k + kvh * a.ks1;
  const uint8_t* vh = a.v + kvh * a.vs1;
  auto fetch = [&](int u) { return fp4_pages<BS>(bt, table_row, bts1, i64 >> 1, a.width, 32 * u, u < end); };
  Fp4Unit<D> ra, rb;
  if (u >= end) pages = fetch(u);
  fp4_load_unit<BS, D, NT>(a, kh, vh, pages, c, g, ra);
  pages = fetch(u + W);
  const Fp4Query<T, D> q = fp4_query<T, D>(query, a.sign, lane);
  WaveState<D> st;
#pragma unroll
  for (int n = 0; n < D / 16; ++n) st.acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  st.m = -INFINITY;
  st.l = 0.f;
  auto step = [&](Fp4Unit<D>& now, Fp4Unit<D>& ahead) -> bool {
    fp4_load_unit<BS, D, NT>(a, kh, vh, pages, c, g, ahead);
    pages = fetch(u + 2 * W);
    fp4_process<T, D>(now, q, a.scale_log2, 32 * u, len - 1, g, st);
    u += W;
    return u < end;
  };
  if (u < end)
    while (step(ra, rb) && step(rb, ra)) {
    }

  // the waves' states meet in LDS; thread -> (head, N dims)
  constexpr int N = D == 128 ? 8 : 4;
  static_assert(64 * W == 16 * (D / N), "a thread for each");
  constexpr int kSpread = acc_spread<D>();
  const int h = threadIdx.x / (D / N), d0 = (threadIdx.x % (D / N)) * N;
  const float lt = column_sum(st.l);
  if (g == 0) {
    s_m[wave][c] = st.m;
    s_l[wave][c] = lt;
  }
#pragma unroll
  for (int rr = 0; rr < 4; ++rr) {
    float* dst = s_acc + (wave * 16 + c) * P + kSpread * ((D / 4) * g + (D / 16) * rr);
    *reinterpret_cast<f32x4*>(dst) = f32x4{st.acc[0][rr], st.acc[1][rr], st.acc[2][rr], st.acc[3][rr]};
    if constexpr (D == 128)
      *reinterpret_cast<f32x4*>(dst + 4) = f32x4{st.acc[4][rr], st.acc[5][rr], st.acc[6][rr], st.acc[7][rr]};
  }
  __syncthreads();
  if (head0 + h >= a.group) return;
  float M = -INFINITY, L = 0.f;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < W; ++x) M = fmaxf(M, s_m[x][h]);
  const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int x = 0; x < W; ++x) {
    const float wt = exp2_fast(s_m[x][h] - mu);
    L += wt * s_l[x][h];
    const float* from = s_acc + (x * 16 + h) * P + kSpread * d0;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] += wt * from[j];
  }
  const int64_t qh = static_cast<int64_t>(kvh) * a.group + head0 + h;
  if (chunks == 1) {
    const float inv = L == 0.f ? 0.f : rcp_fast(L);
    T* dst = static_cast<T*>(a.out) + b * a.os0 + qh * a.os1 + d0 * a.os2;
    if (a.out_rows) {
      const u32x2 lo{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
      if constexpr (N == 8)
        *reinterpret_cast<u32x4*>(dst) =
            u32x4{lo[0], lo[1], pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv)};
      else
        *reinterpret_cast<u32x2*>(dst) = lo;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) dst[j * a.os2] = from_f32<T>(o[j] * inv);
    }
  } else {
    const int64_t at = (static_cast<int64_t>(b) * a.hq + qh) * chunks + chunk;
    float* dst = a.acc + at * D + d0;
    *reinterpret_cast<f32x4*>(dst) = f32x4{o[0], o[1], o[2], o[3]};
    if constexpr (N == 8) *reinterpret_cast<f32x4*>(dst + 4) = f32x4{o[4], o[5], o[6], o[7]};
    if (d0 == 0) a.stats[at] = float2{M, L};
  }
}

// ========================================================== host glue ====
namespace {

int check_decode(const fd_fp4_decode_args* args, const char* fn) {
  if (args == nullptr) return set_error(FD_E_INVALID, "%s: args is NULL", fn);
  const fd_fp4_decode_args& a = *args;
  if (a.struct_size != sizeof(fd_fp4_decode_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, a.struct_size,
                     sizeof(fd_fp4_decode_args));
  if (a.dtype != FD_DTYPE_F16 && a.dtype != FD_DTYPE_BF16)
    return set_error(FD_E_UNSUPPORTED, "%s: dtype must be float16 or bfloat16", fn);
  const int rc = check_fp4_caches(fn, a.head_dim, a.block_size, a.num_blocks, a.num_kv_heads, a.k_cache,
                                  a.k_cache_stride, a.v_cache, a.v_cache_stride);
  if (rc != FD_OK) return rc;
  if (a.num_seqs <= 0 || a.num_q_heads <= 0 || a.max_blocks_per_seq <= 0)
    return set_error(FD_E_INVALID, "%s: shapes must be positive", fn);
  if (a.num_q_heads % a.num_kv_heads != 0)
    return set_error(FD_E_INVALID, "%s: num_q_heads must be divisible by num_kv_heads", fn);
  if (!a.q || !a.block_tables || !a.seq_lens || !a.out) return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (a.seq_lens_stride < 0 || a.seq_lens_stride > INT32_MAX)
    return set_error(FD_E_UNSUPPORTED, "%s: seq_lens stride does not fit 32 bits", fn);
  if (a.max_blocks_per_seq > INT32_MAX || a.max_blocks_per_seq * a.block_size > INT32_MAX - 4096)
    return set_error(FD_E_UNSUPPORTED, "%s: block tables hold 2^31 tokens or more", fn);
  if ((a.kv_reuse != 0 && a.kv_reuse != 1) || (a.ragged != 0 && a.ragged != 1))
    return set_error(FD_E_INVALID, "%s: kv_reuse and ragged must be 0 or 1", fn);
  // (the grid's dimensions: KV heads, rows; a row's head blocks times its chunks)
  if (a.num_seqs > 65535 || a.num_q_heads > (1 << 24))
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

struct Fp4Plan {
  int64_t head_blocks, chunks, chunk_tiles;
  int64_t items, per_cu, floor, least;  // items > 0: chunks by the rows' lengths, at most `chunks` a row
  int64_t acc, stats, live;   // floats
  int64_t floats() const { return acc + stats + live; }
};

// Chunks of rows of `tiles` tiles, `wgs` workgroups a chunk.  In tiles of the time in which
// a CU reads one: the whole call takes at least its average a CU; a CU that has w
// workgroups four fifths of theirs (alone it reads faster than all of them at once); a
// workgroup alone a quarter more than its tiles; and the start and end of one is worth
// four or five, the join of several about 24.  Long tables may be filled unevenly, and short chunks
// come out even: of the counts within a sixteenth of the least the largest.
// MI355X, 128-dim heads, us a call at tiles a chunk, * the nearest to the choice:
//   512 workgroups of 256 tiles: 32 103, 64 96, 128 93, 256 88*, rows from half of that on
//     80, 82, 81, 73*; 256 of 128: 32 30.3, 64 27.6*, 128 25.4; 128 of 1024: 24 105, 48 102*,
//     64 102, 128 106, 256 95;
//   160 of 128: 12 23.6, 24 22.2, 48 20.1*, 128 23.6; 128 of 64: 8 15.7, 16 12.7*, 32 12.4;
//   16 of 64: 2 9.4, 4 7.7*, 8 8.1, 16 9.2; 8 of 256: 4 9.5, 8 8.1*, 16 9.2;
//   2 of 1024: 4 12.9, 8 9.5*, 16 9.3, 64 16.4.
// 64-dim heads, fp16, 32 of 1024 (probabilities in two terms, as above): 12 27.3, 24 24.4,
//   32 22.2*, 64 27.5, rows from 1 / 256 on 14.4, 17.4, 17.3, 21.2.
int64_t chunks_for(int64_t wgs, int64_t tiles, int64_t cus) {
  // (a thread's calls mostly repeat: the last answer is kept)
  static thread_local int64_t last[4] = {0, 0, 0, 0};
  if (last[0] == wgs && last[1] == tiles && last[2] == cus) return last[3];
  auto counts = [&](auto take) {
    for (int64_t n = 1; n == 1 || (n * wgs <= 16 * cus && 2 * n <= tiles + 1); ++n) {
      const int64_t per = (tiles + n - 1) / n, w = (n * wgs + cus - 1) / cus;
      double cost = static_cast<double>(wgs) * tiles / cus;
      cost = cost > 0.8 * w * per ? cost : 0.8 * w * per;
      cost = cost > 1.25 * per ? cost : 1.25 * per;
      take(n, cost + 4.5 * w + (n > 1 ? 24 : 0));
    }
  };
  double least = 1e300;
  int64_t best = 1;
  counts([&](int64_t n, double cost) {
    if (cost < least) {
      least = cost;
      best = n;
    }
  });
  if (best > 1 && tiles >= 256) counts([&](int64_t n, double cost) { best = 16 * cost <= 17 * least ? n : best; });
  last[0] = wgs;
  last[1] = tiles;
  last[2] = cus;
  return last[3] = best;
}

Fp4Plan plan_for(const fd_fp4_decode_args& a) {
  Fp4Plan s{};
  s.head_blocks = (a.num_q_heads / a.num_kv_heads + 15) / 16;
  const int64_t tiles = (a.max_blocks_per_seq * a.block_size + 31) / 32;
  const int64_t wgs = a.num_seqs * a.num_kv_heads * s.head_blocks;
  const int64_t chunks = chunks_for(wgs, tiles, device_cus());
  s.chunk_tiles = (tiles + chunks - 1) / chunks;
  s.chunks = (tiles + s.chunk_tiles - 1) / s.chunk_tiles;
  // By the rows' lengths where a table's width would cut rows too, they are few enough and
  // CUs have enough to read to pay for finding the chunks (1 us), or where the caller says
  // that the lengths differ widely.  128-dim heads bf16, us a call, by width / by lengths of
  // rows from 1 / 256 of the table on, from half of it, full: 16 x 8 pairs of 1024 tiles
  // 34.1 / 25.0, 80 / 75, 101 / 92; 8 x 8 of 256 12.3 / 9.4, 18.6 / 15.6, 19.8 / 17.3; 32 x 8
  // of 256 24.6 / 16.7, 45.4 / 41.6, 51.4 / 50.5; 32 x 2 of 256 13.4 / 10.0, 19.1 / 16.5, 21.4 / 18.0;
  // 128 x 2 of 256 26.6 / 19.7, 52.1 / 46.3, 55.2 / 54.2.  In shorter tables even rows lose what
  // uneven ones gain a few times over: 64 x 2 of 128 13.5 / 11.2, 16.5 / 16.4, 17.8 / 18.5, of 64
  // 11.3 / 10.0, 12.5 / 12.8, 12.6 / 13.1; 32 x 8 of 128 18.2 / 13.4, 24.8 / 26.9, 27.8 / 29.8; in the
  // shortest all do (probabilities in one term: 8 x 2 of 64 7.3 / 7.7, -, 7.8 / 8.2).
  // Where the width does not cut, so only if asked for: 64 x 8 of 1024 152 / 79, 282 / 280,
  // 345 / 351, of 256 43 / 28, 73 / 80, 88 / 97; 128 x 8 of 256 51 / 51, 136 / 155, 172 / 190.  64-dim
  // heads fp16, 16 x 2 of 1024 14.2 / 11.0, 22.2 / 19.6, 23.5 / 22.4.
  // Two chunks a CU of 16 tiles or more for few pairs (four take 0 to 8 % more), four of 32
  // where each CU has a pair (32 x 8 of 256: 17.2, 41.9, 50.2; two 19.0, 44.3, 50.3; eight 16.7,
  // 43.2, 52.3), eight for two, and so on.
  // Chunks a row has room for: 16, which the join takes with a wave a row (more cost 32 x 8 of
  // 256 4 us), and so many that a wide table's are no longer than 64 tiles (16 x 8 rows of
  // 8192 tokens in tables of 131072: 45 us with 16 chunks, 30 with 64, 31 in tables of 8192;
  // rows of 2048 16.6, 17.6, 13.3); few pairs, whose partials are small, 32 times their share
  // (8 x 2 rows of 2048 in such tables: 128 chunks 12.1, 256 8.2; 7.8 in their own).
  const int64_t cus = device_cus();
  // (of 32 tiles on: a row of a table that is one chunk has no join to write it)
  if ((s.chunks > 1 || a.ragged) && a.num_seqs <= kFp4ItemRows && tiles >= 32 && wgs * tiles >= 16 * cus &&
      a.num_seqs * tiles < (1 << 30)) {
    const bool few = 2 * wgs <= cus;
    s.per_cu = few ? 2 : 4 * ((wgs + cus - 1) / cus);
    s.floor = few ? 16 : 32;
    s.items = std::max(s.per_cu * cus / (a.num_kv_heads * s.head_blocks), 2 * a.num_seqs);
    const int64_t share = s.items / a.num_seqs;
    const int64_t most = share <= 8 ? std::min(std::max(tiles / 64, int64_t{16}), int64_t{128})
                                    : std::min(32 * share, int64_t{1024});
    s.least = std::max((tiles + most - 1) / most, int64_t{4});
    s.chunks = std::min(s.items, (tiles + s.least - 1) / s.least);
  }
  if (s.chunks > 1) {
    const int64_t rows = a.num_seqs * a.num_q_heads;
    s.acc = rows * s.chunks * a.head_dim;
    s.stats = (2 * rows * s.chunks + 3) & ~int64_t{3};
    s.live = s.items > 0 ? a.num_seqs : 0;
  }
  return s;
}

int check_plan(const fd_fp4_decode_args& a, const Fp4Plan& s, const char* fn) {
  if (!grid_fits((s.chunks + 1) * s.head_blocks, 64 * kFp4Waves) || a.num_seqs * a.num_q_heads > INT32_MAX)
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

bool rows_on_lines(const void* at, const int64_t* stride) {
  return stride[2] == 1 && stride[0] % 8 == 0 && stride[1] % 8 == 0 && (reinterpret_cast<uintptr_t>(at) & 15u) == 0;
}

template <typename T, int D>
void launch_decode(const fd_fp4_decode_args& a, const Fp4Plan& s, const Fp4Args& p, hipStream_t stream) {
  // (many chunks of more than one round: an odd number, the last of which may be none, so
  // that those which short rows do not have are spread over the XCDs; 16 rows of 128 ..
  // 32768 tokens, Hq 32, Hkv 8, 16 / 17 chunks: 49 / 32 us, by their lengths 25)
  const bool rounds = a.num_seqs * a.num_kv_heads * s.chunks * s.head_blocks > device_cus();
  const int64_t per_row = s.items > 0 ? 1 : s.chunks | (rounds && s.chunks >= 8 ? 1 : 0);
  const dim3 grid(static_cast<unsigned>(per_row * s.head_blocks), static_cast<unsigned>(a.num_kv_heads),
                  static_cast<unsigned>(s.items > 0 ? s.items : a.num_seqs));
  const int i64 = (a.seq_lens_dtype == FD_INDEX_I64 ? 1 : 0) | (a.block_tables_dtype == FD_INDEX_I64 ? 2 : 0);
  auto go = [&](auto kernel) {
    dispatch(kernel, grid, dim3(64 * kFp4Waves), stream, nullptr, nullptr, a.seq_lens, a.block_tables,
             a.block_tables_stride[0], a.block_tables_stride[1], static_cast<int32_t>(a.seq_lens_stride), i64,
             static_cast<int32_t>(s.chunks), static_cast<int32_t>(s.chunk_tiles), p);
  };
  const bool nt = a.kv_reuse == 0;
  switch (a.block_size) {
    case 8: nt ? go(fp4_decode_kernel<T, 8, D, true>) : go(fp4_decode_kernel<T, 8, D, false>); break;
    case 16: nt ? go(fp4_decode_kernel<T, 16, D, true>) : go(fp4_decode_kernel<T, 16, D, false>); break;
    default: nt ? go(fp4_decode_kernel<T, 32, D, true>) : go(fp4_decode_kernel<T, 32, D, false>); break;
  }
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_fp4_decode_floats(const fd_fp4_decode_args* args, int64_t* floats) {
  static const char* fn = "fd_fp4_decode_floats";
  const int rc = check_decode(args, fn);
  if (rc != FD_OK) return rc;
  if (floats == nullptr) return set_error(FD_E_INVALID, "%s: floats is NULL", fn);
  *floats = plan_for(*args).floats();
  return FD_OK;
}

extern "C" int fd_fp4_decode(const fd_fp4_decode_args* args, float* workspace, int64_t floats, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_fp4_decode";
  int rc = check_decode(args, fn);
  if (rc != FD_OK) return rc;
  const fd_fp4_decode_args& a = *args;
  const Fp4Plan s = plan_for(a);
  rc = check_plan(a, s, fn);
  if (rc != FD_OK) return rc;
  if (s.floats() > 0 && (workspace == nullptr || floats < s.floats() || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return set_error(FD_E_INVALID, "%s: needs a 16-byte aligned workspace of %lld floats", fn,
                     static_cast<long long>(s.floats()));
  Fp4Args p{};
  p.q = a.q;
  p.k = static_cast<const uint8_t*>(a.k_cache);
  p.v = static_cast<const uint8_t*>(a.v_cache);
  p.out = a.out;
  p.acc = workspace;
  p.stats = reinterpret_cast<float2*>(workspace + s.acc);
  p.live = reinterpret_cast<int32_t*>(workspace + s.acc + s.stats);
  p.rows = static_cast<int>(a.num_seqs);
  p.items = static_cast<int>(s.items);
  p.per_cu = static_cast<int>(s.per_cu);
  p.floor = static_cast<int>(s.floor);
  p.least = static_cast<int>(s.least);
  p.qs0 = a.q_stride[0];
  p.qs1 = a.q_stride[1];
  p.qs2 = a.q_stride[2];
  p.ks0 = a.k_cache_stride[0];
  p.ks1 = a.k_cache_stride[1];
  p.vs0 = a.v_cache_stride[0];
  p.vs1 = a.v_cache_stride[1];
  p.os0 = a.out_stride[0];
  p.os1 = a.out_stride[1];
  p.os2 = a.out_stride[2];
  p.q_rows = rows_on_lines(a.q, a.q_stride);
  p.out_rows = rows_on_lines(a.out, a.out_stride);
  p.hq = static_cast<int>(a.num_q_heads);
  p.group = static_cast<int>(a.num_q_heads / a.num_kv_heads);
  p.head_blocks = static_cast<int>(s.head_blocks);
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.width = static_cast<int>(a.max_blocks_per_seq);
  p.wide = a.block_tables_dtype == FD_INDEX_I64 ? -1 : 0;
  p.cap = static_cast<int>(a.max_blocks_per_seq * a.block_size);
  const float scale = a.sm_scale * kLog2e;
  p.sign = scale > 0.f ? 1.f : (scale < 0.f ? -1.f : scale);
  p.scale_log2 = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const bool bf = a.dtype == FD_DTYPE_BF16;
  if (a.head_dim == 64)
    bf ? launch_decode<__bf16, 64>(a, s, p, stream) : launch_decode<_Float16, 64>(a, s, p, stream);
  else
    bf ? launch_decode<__bf16, 128>(a, s, p, stream) : launch_decode<_Float16, 128>(a, s, p, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  if (s.chunks == 1) return FD_OK;
  RowJoin j{};
  j.acc = p.acc;
  j.stats = p.stats;
  j.seq_lens = a.seq_lens;
  j.seq_lens_stride = a.seq_lens_stride;
  j.seq_lens_i64 = a.seq_lens_dtype == FD_INDEX_I64;
  j.hkv = static_cast<int>(a.num_kv_heads);
  j.group = p.group;
  j.chunks = static_cast<int>(s.chunks);
  j.chunk_tiles = static_cast<int>(s.chunk_tiles);
  j.cap = p.cap;
  j.rows = a.num_seqs * a.num_q_heads;
  if (s.items > 0) {  // as rows of as many tiles as they have chunks
    j.seq_lens = p.live;
    j.seq_lens_stride = 1;
    j.seq_lens_i64 = false;
    j.chunk_tiles = 1;
    j.cap = static_cast<int>(32 * s.chunks);
  }
  j.out = a.out;
  for (int i = 0; i < 3; ++i) j.out_stride[i] = a.out_stride[i];
  return join_rows(j, bf, static_cast<int>(a.head_dim), fn, stream);
}
