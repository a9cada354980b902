// Decode attention of a bounded cache, for gfx950.
//
//   window: the query attends the row's first `sinks` tokens and its last
//           `window` ones.
//   scored: the query attends every token, and the weight that each token
//           receives from the query heads of its KV head is added to a table.
//
// With s = scale * q.k, the softmax over a row's attended tokens A is
//   out = sum_A 2^(x_t - M) v_t / L,  x = s log2(e), M = max x, L = sum 2^(x - M).
// A row's tiles (bounded_row.h) are cut into chunks of the same length, one per
// workgroup; each leaves (M, L, sum 2^(x - M) v) of its chunk, and a second launch
// joins them: out = sum_c 2^(M_c - M) acc_c / sum_c 2^(M_c - M) L_c.  A token's
// weight needs the whole row's M and L, so a scored chunk also leaves its x
// (4 bytes a query head, next to 4 D bytes of K and V a KV head), from which the
// second launch forms sum_h 2^(x_h - M_h - log2 L_h).  Short scored rows, and rows
// enough for the card, are one workgroup's each and need no second launch.
#include "decode_host.h"
#include "bounded_row.h"
#include "dim_major_unit.h"

namespace fd {

struct BoundedParams {
  int window, sinks;
  int chunk_tiles, chunks;  // tiles of a chunk; chunks of a row at most
  int units;                // 16-token units of a full table row
  float* acc;               // [row, chunk, D] (row: request, query head)
  float2* stats;            // [row, chunk] (M, L)
  float* raw;               // [pair, raw_at] x of every token, scored only
  float* scores;            // [request, KV head, token], scored only
  int64_t scs0, scs1;
  bool ragged;              // lengths vary widely, scored only
};

__device__ __forceinline__ BoundedRow bounded_row_of(const DecodeParams& p, const BoundedParams& w, int b) {
  const int cap = static_cast<int>(p.max_blocks_per_seq * p.block_size);
  return bounded_row(load_index(p.sl, b * p.sls, p.sl_i64), cap, w.window, w.sinks);
}

// Float of token t (of the row) and head h of the group within a pair's scores.
__device__ __forceinline__ int64_t raw_at(int t, int h, int group) {
  return (static_cast<int64_t>(t >> 2) * group + h) * 4 + (t & 3);
}

// Weight of a token with score x in a row with M + log2 L = z (infinity: a row that
// attends nothing).  ODD: z may be NaN, where the row's scores hold a NaN or +inf: so is
// every weight of the row, but a token that is not attended (-inf) has none.  Asked once
// for all heads: a comparison a weight costs a chat's call 0.4 of 10.8 us.
template <bool ODD>
__device__ __forceinline__ float token_weight(float x, float z) {
  const float w = exp2_fast(x - z);
  return ODD && x == -INFINITY ? 0.f : w;
}
__device__ __forceinline__ bool any_nan(const float* z, int n) {  // of up to 64, by the whole wave
  const float mine = z[min(static_cast<int>(threadIdx.x & 63), n - 1)];
  return __ballot(mine != mine) != 0;
}

// ====================================================== any strides ======
// One wave per (request, KV head, up to 8 query heads, chunk): caches of any
// layout, alignment and group size, element by element.  Lane = token for q.k,
// lane = dim for the weighted sum.
constexpr int kBoundedHeads = 8;

template <typename T, int D, bool SCORED>
__global__ __launch_bounds__(64) void bounded_generic_kernel(DecodeParams p, BoundedParams w, int head_groups) {
  __shared__ float s_q[kBoundedHeads][D];
  __shared__ float s_p[kBoundedHeads][64];
  __shared__ int64_t s_vrow[64];  // element offset of the V row, -1: masked

  const int lane = threadIdx.x;
  const int chunk = blockIdx.y / head_groups;
  const int hg = blockIdx.y % head_groups;
  const int pair = blockIdx.x;
  const int b = pair / p.hkv;
  const int kvh = pair % p.hkv;
  const int h0 = hg * kBoundedHeads;  // within the group
  const int nh = min(kBoundedHeads, p.group - h0);
  const BoundedRow r = bounded_row_of(p, w, b);
  const int t_begin = chunk * w.chunk_tiles, t_end = min(t_begin + w.chunk_tiles, r.tiles);
  if (t_begin >= t_end && w.chunks > 1) return;  // the join reads a row's own chunks only

  const T* qb = static_cast<const T*>(p.q) + b * p.qs0;
  for (int i = lane; i < kBoundedHeads * D; i += 64) {
    const int j = i / D, d = i % D;
    s_q[j][d] = j < nh ? to_f32(qb[(kvh * p.group + h0 + j) * p.qs1 + d * p.qs2]) : 0.f;
  }
  const T* kbase = static_cast<const T*>(p.k);
  const T* vbase = static_cast<const T*>(p.v);
  float m[kBoundedHeads], l[kBoundedHeads], acc[kBoundedHeads][D / 64];
#pragma unroll
  for (int j = 0; j < kBoundedHeads; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) acc[j][e] = 0.f;
  }
  __syncthreads();

  for (int i0 = t_begin; i0 < t_end; i0 += 2) {  // two tiles, one token a lane
    const int i = i0 + (lane >> 5);
    const int tok = 32 * r.tile(i) + (lane & 31);
    bool ok = i < t_end && r.attends(tok);
    int64_t krow = 0, vrow = -1;
    if (ok) {
      const int64_t blk = load_index(p.bt, b * p.bts0 + (tok / p.block_size) * p.bts1, p.bt_i64);
      ok = blk >= 0 && blk < p.num_blocks;
      const int64_t off = tok % p.block_size;
      krow = blk * p.ks0 + kvh * p.ks1 + off * p.ks2;
      vrow = ok ? blk * p.vs0 + kvh * p.vs1 + off * p.vs2 : -1;
    }
    float sc[kBoundedHeads];
#pragma unroll
    for (int j = 0; j < kBoundedHeads; ++j) sc[j] = 0.f;
    if (ok) {
      for (int d = 0; d < D; ++d) {
        const float kv = to_f32(kbase[krow + d * p.ks3]);
#pragma unroll
        for (int j = 0; j < kBoundedHeads; ++j) sc[j] += s_q[j][d] * kv;
      }
    }
    s_vrow[lane] = vrow;
#pragma unroll
    for (int j = 0; j < kBoundedHeads; ++j) {
      const float s = ok ? sc[j] * p.scale_log2 : -INFINITY;
      if (SCORED && j < nh && i < t_end)
        w.raw[static_cast<int64_t>(pair) * w.units * p.group * 16 + raw_at(tok, h0 + j, p.group)] = s;
      float mx = s;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, shfl_xor_f32(mx, o));
      const float m_new = fmaxf(m[j], mx);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[j] - m_use);
      const float pj = exp2f(s - m_use);
      float ps = pj;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) ps += shfl_xor_f32(ps, o);
      l[j] = l[j] * alpha + ps;
      m[j] = m_new;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) acc[j][e] *= alpha;
      s_p[j][lane] = pj;
    }
    __syncthreads();
    for (int t = 0; t < 64; ++t) {
      const int64_t vr = s_vrow[t];
      if (vr < 0) continue;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        const float vv = to_f32(vbase[vr + (lane + 64 * e) * p.vs3]);
#pragma unroll
        for (int j = 0; j < kBoundedHeads; ++j) acc[j][e] += s_p[j][t] * vv;
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int j = 0; j < kBoundedHeads; ++j) {
    if (j >= nh) break;
    const int qh = kvh * p.group + h0 + j;
    if (!SCORED && w.chunks == 1) {
      const float inv = l[j] > 0.f ? 1.f / l[j] : 0.f;
      T* dst = static_cast<T*>(p.out) + b * p.os0 + qh * p.os1;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) dst[(lane + 64 * e) * p.os2] = from_f32<T>(acc[j][e] * inv);
    } else {
      const int64_t at = (static_cast<int64_t>(b) * p.hq + qh) * w.chunks + chunk;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) w.acc[at * D + lane + 64 * e] = acc[j][e];
      if (lane == 0) w.stats[at] = float2{m[j], l[j]};
    }
  }
}

// ===================================================== MFMA kernel =======
// Token-major caches with 16-byte rows: one workgroup of W waves per (request, KV
// head, 16 NCB query heads, chunk), its waves taking 16-token units in turn.
// A unit's K/V are in registers (UnitRegs), the next unit's on their way and the
// block id after it being read.  Large calls are bound by HBM reads: 64 rows of a
// 4096-token window and 64 sinks, Hq 32, Hkv 8, D 128, one chunk a row: 1.09 GB in
// 160 us, 6.8 TB/s; 32 scored rows of 4096 .. 8192 tokens, whole: 0.82 GB in 147 us,
// 5.6 TB/s, the longest rows last.  Small ones by their start, three dependent loads
// (length, block id, K/V), and by the join.
constexpr int kBoundedWaves = 4;
constexpr int kBoundedUnit = 16;
// What a workgroup does with its rows' end: window chunks and whole rows, scored
// chunks, and whole scored rows, whose scores stay in LDS.
enum BoundedMode { kWindow, kScored, kScoredWhole };
constexpr int kWholeWaves = 4;

// Launch arguments, strides in elements; the host checks that they fit.
struct BoundedArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* bt;
  const void* sl;
  void* out;
  float* acc;
  float2* stats;
  float* raw;
  float* scores;
  int64_t scs0, scs1;
  // (ks2, vs2: between a block's rows, which are tokens, or dims of dim-major caches)
  int32_t qs0, qs1, ks0, ks1, ks2, vs0, vs1, vs2, bts0, bts1, sls, os0, os1, os2;
  int32_t out_rows;  // out's rows have unit stride and lie on 16-byte lines
  int32_t i64;  // bit 0: 64-bit lengths, bit 1: 64-bit block tables
  int32_t num_blocks, hkv, hq, group, cap, width;
  int32_t window, sinks, chunk_tiles, chunks, units;
  float scale_log2;
};

// A unit's block ids, -1 past the chunk's last unit.
struct BoundedPages {
  int32_t a, b;  // b: blocks of 8 tokens only
};

template <int BS>
__device__ __forceinline__ BoundedPages bounded_pages(const BoundedArgs& a, int64_t table_row, int tok0, bool live) {
  BoundedPages p{-1, -1};
  if (!live) return p;
  const int first = tok0 / BS;
  p.a = load_index_uniform(a.bt, table_row + static_cast<int64_t>(first) * a.bts1, a.i64 >> 1);
  // (a row's last unit may end behind its table)
  if constexpr (BS == 8)
    p.b = load_index_uniform(a.bt, table_row + static_cast<int64_t>(min(first + 1, a.width - 1)) * a.bts1, a.i64 >> 1);
  return p;
}

// One 16- or 8-byte piece of a K/V row through a descriptor (aux 2: streamed
// past the caches); an empty descriptor reads nothing and gives zeros.
template <bool NT, typename V>
__device__ __forceinline__ V bounded_load_piece(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff) {
  if constexpr (sizeof(V) == 16)
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voff, soff, NT ? 2 : 0));
  else
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(rsrc, voff, soff, NT ? 2 : 0));
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t bounded_rsrc(const char* at, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at), 0, bytes, 0x00020000);
}

// A unit's K and V.  Blocks of 16 and 32 tokens: the unit lies in one, so its
// rows are a descriptor at the block (uniform) plus the lane's offset.  Blocks of
// 8: the lane's half picks the block.  As many loads are issued for a unit that is
// not there, so that the wait for the unit before never covers them.
template <typename T, int BS, int D, bool NT>
__device__ __forceinline__ void bounded_load(const BoundedArgs& a, const char* kh, const char* vh,
                                             const BoundedPages& p, int row0, int c, int g,
                                             UnitRegs<kBoundedUnit, D>& t) {
  constexpr int E = sizeof(T);
  constexpr int KS = D / 32;
  const uint32_t ks2 = a.ks2, vs2 = a.vs2;
  if constexpr (BS >= 16) {
    // -1 for a valid block, else 0, by integer arithmetic (opaque in the middle: as a
    // comparison's result the compiler selects it in a vector register, and every
    // load becomes a loop over its descriptor's lanes)
    int past = p.a - a.num_blocks;
    asm("" : "+s"(past));
    const int ok = (past & ~p.a) >> 31;
    const int64_t blk = p.a & ok;
    const __amdgpu_buffer_rsrc_t kr = bounded_rsrc(kh + blk * a.ks0 * E, ok);
    const __amdgpu_buffer_rsrc_t vr = bounded_rsrc(vh + blk * a.vs0 * E, ok);
    const uint32_t ko = (c * ks2 + 8 * g) * E, vo = (4 * g * vs2 + (D / 16) * c) * E;
#pragma unroll
    for (int s = 0; s < KS; ++s) t.kf[0][s] = bounded_load_piece<NT, u32x4>(kr, ko + 64 * s, row0 * ks2 * E);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.vf[i] = bounded_load_piece<NT, VPiece<D>>(vr, vo, (row0 + i) * vs2 * E);
    t.bmask = static_cast<uint32_t>(ok) & 0xfu;
  } else {
    const int32_t kpage = c < 8 ? p.a : p.b, vpage = g < 2 ? p.a : p.b;
    const bool kok = kpage >= 0 && kpage < a.num_blocks, vok = vpage >= 0 && vpage < a.num_blocks;
    // rows of no block read the start of the cache: one line
    const char* kp = kok ? kh + (static_cast<int64_t>(kpage) * a.ks0 + static_cast<int64_t>(c & 7) * a.ks2 + 8 * g) * E
                         : static_cast<const char*>(a.k);
    const char* vp = vok ? vh + (static_cast<int64_t>(vpage) * a.vs0 + static_cast<int64_t>(4 * (g & 1)) * a.vs2 + (D / 16) * c) * E
                         : static_cast<const char*>(a.v);
    const int64_t vstep = vok ? static_cast<int64_t>(a.vs2) * E : 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) t.kf[0][s] = kv_load<NT>(kp + 64 * s);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.vf[i] = kv_load<NT, VPiece<D>>(vp + i * vstep);
    t.bmask = vok ? 0xfu : 0u;
  }
}

// The same for a 32-token unit of a dim-major cache (load_unit_dm's layout).  Blocks
// of 32 tokens hold a unit, the others a quarter or a half: the lane's eight tokens
// pick the block.
template <int BS>
__device__ __forceinline__ UnitPages bounded_pages_dm(const BoundedArgs& a, int64_t table_row, int tok0, bool live) {
  UnitPages p{-1, -1, -1, -1};
  if (!live) return p;
  auto entry = [&](int i) {
    const int at = min(tok0 / BS + i, a.width - 1);
    return load_index_uniform(a.bt, table_row + static_cast<int64_t>(at) * a.bts1, a.i64 >> 1);
  };
  p.a = entry(0);
  if constexpr (BS <= 16) p.b = entry(1);
  if constexpr (BS == 8) {
    p.c = entry(2);
    p.d = entry(3);
  }
  return p;
}

template <typename T, int BS, int D, bool NT>
__device__ __forceinline__ void bounded_load_dm(const BoundedArgs& a, const char* kh, const char* vh, const UnitPages& p,
                                                int lane, DmRegs<D>& t) {
  constexpr int E = sizeof(T), KS = DmRegs<D>::KS;
  const int q = lane & 3, c = lane & 15, g = lane >> 4;
  const uint32_t ks = a.ks2, vs = a.vs2;
  if constexpr (BS == 32) {
    int past = p.a - a.num_blocks;
    asm("" : "+s"(past));
    const int ok = (past & ~p.a) >> 31;
    const int64_t blk = p.a & ok;
    const __amdgpu_buffer_rsrc_t kr = bounded_rsrc(kh + blk * a.ks0 * E, ok);
    const __amdgpu_buffer_rsrc_t vr = bounded_rsrc(vh + blk * a.vs0 * E, ok);
    const uint32_t ko = ((lane >> 2) * ks + 8 * q) * E, vo = (c * vs + 8 * g) * E;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      t.kf[i / KS][i % KS] = bounded_load_piece<NT, u32x4>(kr, ko, 16 * i * ks * E);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) t.vf[n] = bounded_load_piece<NT, u32x4>(vr, vo, 16 * n * vs * E);
    t.bmask = static_cast<uint32_t>(ok) & 0xffu;
  } else {
    auto page = [&](int x) {
      if constexpr (BS == 16) return x < 2 ? p.a : p.b;
      return x == 0 ? p.a : x == 1 ? p.b : x == 2 ? p.c : p.d;
    };
    const int32_t kpage = page(q), vpage = page(g);
    const bool kok = kpage >= 0 && kpage < a.num_blocks, vok = vpage >= 0 && vpage < a.num_blocks;
    // pieces of no block read the start of the cache: one line
    const char* kp = kok ? kh + (static_cast<int64_t>(kpage) * a.ks0 + static_cast<int64_t>(lane >> 2) * ks + (8 * q) % BS) * E
                         : static_cast<const char*>(a.k);
    const char* vp = vok ? vh + (static_cast<int64_t>(vpage) * a.vs0 + static_cast<int64_t>(c) * vs + (8 * g) % BS) * E
                         : static_cast<const char*>(a.v);
    const int64_t kstep = kok ? 16ll * ks * E : 0, vstep = vok ? 16ll * vs * E : 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) t.kf[i / KS][i % KS] = kv_load<NT>(kp + i * kstep);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) t.vf[n] = kv_load<NT>(vp + n * vstep);
    t.bmask = vok ? 0xffu : 0u;
  }
}

// Leaves a unit's scores for the weights: lane (c, g) holds tokens 4g .. 4g + 3 of
// head c, and the unit is laid out [g][head of the group][4 tokens], so that
// neighbouring lanes fill a 64-byte piece.  The store goes through a descriptor
// that drops the columns behind the group: under a branch the compiler no longer
// knows how many memory operations are in flight, and waits for the next unit's
// loads before it uses this one's.
template <int NCB>
struct KeepScores {
  __amdgpu_buffer_rsrc_t unit;
  uint32_t at[NCB];  // this lane's byte in the unit; past its end: no such head
  template <int VR>
  __device__ __forceinline__ void operator()(int cb, const float (&sc)[VR]) const {
    const f32x4 x{sc[0], sc[1], sc[2], sc[3]};
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), unit, at[cb], 0, 0);
  }
};

// The same of a dim-major unit: lane (c, g) holds tokens 8g .. 8g + 7 of head c.
struct KeepScoresDm {
  __amdgpu_buffer_rsrc_t unit;
  uint32_t at, step;  // step: bytes of four tokens
  template <int VR>
  __device__ __forceinline__ void operator()(int, const float (&sc)[VR]) const {
    static_assert(VR == 8);
    const f32x4 x{sc[0], sc[1], sc[2], sc[3]}, y{sc[4], sc[5], sc[6], sc[7]};
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), unit, at, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), unit, at + step, 0, 0);
  }
};

// The same in LDS (scored rows of one workgroup).
struct KeepScoresLds {
  float* unit;
  int at, step;  // this lane's float in the unit, -1: no such head; floats of four tokens
  template <int VR>
  __device__ __forceinline__ void operator()(int, const float (&sc)[VR]) const {
    if (at < 0) return;
#pragma unroll
    for (int i = 0; i < VR / 4; ++i)
      *reinterpret_cast<f32x4*>(unit + at + i * step) = f32x4{sc[4 * i], sc[4 * i + 1], sc[4 * i + 2], sc[4 * i + 3]};
  }
};

// The leading arguments, which the first loads need, are preloaded into SGPRs; the
// others are fetched while the row's length is on its way.
// DM: dim-major caches, in units of 32 tokens (dim_major_unit.h).
template <typename T, int BS, int D, int NCB, int MODE, int W, bool NT, bool DM = false>
__global__ __launch_bounds__(64 * W, 2) void bounded_mfma_kernel(
    const void* sl, const void* bt, int32_t sls, int32_t bts0, int32_t bts1, int32_t hkv, int32_t chunks,
    int32_t chunk_tiles, int32_t cap, int32_t window, int32_t sinks, int32_t i64, BoundedArgs args) {
  constexpr int KS = D / 32;
  constexpr bool SCORED = MODE != kWindow, WHOLE = MODE == kScoredWhole;
  static_assert(!WHOLE || NCB == 1, "whole scored rows: up to 16 heads a KV head");
  static_assert(!DM || NCB == 1, "dim-major: 16 heads a workgroup");
  constexpr int kUnit = DM ? 32 : kBoundedUnit, kUnits = 32 / kUnit;  // tokens of a unit, units of a tile
  // a wave's state of one column block, a head a row (whole scored rows: of the
  // group's heads only, and the row's scores, as raw_at, behind them)
  constexpr int P = acc_pitch<D>();
  __shared__ __attribute__((aligned(16))) float s_fixed[WHOLE ? 4 : W * 16 * P];
  extern __shared__ __attribute__((aligned(16))) float s_more[];
  float* s_acc = WHOLE ? s_more : s_fixed;
  const int acc_rows = WHOLE ? args.group : 16;
  [[maybe_unused]] float* s_raw = s_more + W * acc_rows * P;
  __shared__ float s_m[W][16], s_l[W][16];
  __shared__ float s_z[WHOLE ? 16 : 1];
  // Consecutive workgroups, on one XCD after the other, take a row's chunks, so that a
  // long row's K/V come through all of them.  A grid of more than one round has an odd
  // number of chunks (the last may be none), so that the chunks which short rows do
  // not have are spread over the XCDs too (16 rows of 32 .. 8192 tokens, Hq 32, Hkv 8,
  // eight tiles a chunk: 59.6 us with 32 chunks, 30.6 with 33; one round, eight rows of
  // 2048, Hq 16, Hkv 2, 16 chunks: 10.8, with 17 12.5).
  const int b = blockIdx.z, kvh = blockIdx.y, pair = b * hkv + kvh;
  int chunk = blockIdx.x, hb = 0;
  if constexpr (NCB > 1 || DM) {
    const int hblocks = (args.group + 16 * NCB - 1) / (16 * NCB);
    chunk = blockIdx.x / hblocks;
    hb = blockIdx.x - chunk * hblocks;
  }
  const int len = load_index_uniform(sl, static_cast<int64_t>(b) * sls, i64 & 1);
  BoundedArgs a = args;
  asm volatile("" ::"s"(a.q), "s"(a.k), "s"(a.v), "s"(a.qs0), "s"(a.qs1), "s"(a.ks0), "s"(a.ks1), "s"(a.ks2),
               "s"(a.vs0), "s"(a.vs1), "s"(a.vs2), "s"(a.num_blocks), "s"(a.group), "s"(a.scale_log2));
  a.bt = bt;
  a.bts0 = bts0;
  a.bts1 = bts1;
  a.i64 = i64;
  const int head0 = 16 * NCB * hb;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;

  // Ahead of the K/V loads, so that their number in flight is the same on entry to the
  // loop and in it (waits are for the least of both).  Columns past the group's last
  // head take its first; their results are dropped
  u32x4 qf[NCB][KS];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    const int h = head0 + 16 * cb + c;
    const T* row = static_cast<const T*>(a.q) + static_cast<int64_t>(b) * a.qs0 +
                   static_cast<int64_t>(kvh * a.group + (h < a.group ? h : 0)) * a.qs1;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[cb][s] = *reinterpret_cast<const u32x4*>(row + 32 * s + 8 * g);
  }
  const BoundedRow r = bounded_row(len, cap, window, sinks);
  const int begin = chunk * chunk_tiles, end = min(begin + chunk_tiles, r.tiles);
  if (begin >= end && !WHOLE && (SCORED || chunks > 1)) return;  // the join reads a row's own chunks only
  // (the line's last tile is the row's; its second unit may hold no token)
  const int u_end = kUnits * end - (kUnits == 2 && end == r.tiles && ((r.len - 1) & 31) < 16 ? 1 : 0);
  int u = kUnits * begin + wave;
  const int64_t table_row = static_cast<int64_t>(b) * a.bts0;
  auto token0 = [&](int unit) {
    return DM ? 32 * r.tile(unit) : 32 * r.tile(unit >> 1) + 16 * (unit & 1);
  };
  const char* kh = static_cast<const char*>(a.k) + static_cast<int64_t>(kvh) * a.ks1 * static_cast<int>(sizeof(T));
  const char* vh = static_cast<const char*>(a.v) + static_cast<int64_t>(kvh) * a.vs1 * static_cast<int>(sizeof(T));
  const int row0 = (16 * wave) % BS;  // units advance by whole blocks

  using Regs = std::conditional_t<DM, DmRegs<D>, UnitRegs<kBoundedUnit, D>>;
  auto fetch = [&](int unit) {
    if constexpr (DM)
      return bounded_pages_dm<BS>(a, table_row, token0(unit), unit < u_end);
    else
      return bounded_pages<BS>(a, table_row, token0(unit), unit < u_end);
  };
  Regs ra, rb;
  auto pages = fetch(u);
  auto load = [&](Regs& t) {
    if constexpr (DM)
      bounded_load_dm<T, BS, D, NT>(a, kh, vh, pages, lane, t);
    else
      bounded_load<T, BS, D, NT>(a, kh, vh, pages, row0, c, g, t);
  };
  load(ra);
  pages = fetch(u + W);

  WaveState<D> st[NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n) st[cb].acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    st[cb].m = -INFINITY;
    st[cb].l = 0.f;
  }
  __shared__ __attribute__((aligned(16))) uint8_t s_stage[DM ? W * D * kDmRowBytes : 16];
  [[maybe_unused]] const char* raw =
      reinterpret_cast<const char*>(a.raw + static_cast<int64_t>(pair) * a.units * a.group * 16);
  using Keep = std::conditional_t<DM, KeepScoresDm, KeepScores<NCB>>;
  std::conditional_t<WHOLE, KeepScoresLds, std::conditional_t<SCORED, Keep, NoScores>> keep;
  if constexpr (WHOLE) {
    keep.at = c < a.group ? 4 * (kUnit / 16 * g * a.group + c) : -1;
    keep.step = 4 * a.group;
  } else if constexpr (SCORED && DM) {
    const int h = head0 + c;
    keep.at = h < a.group ? 16u * (2 * g * a.group + h) : 0x7fffffffu;
    keep.step = 16u * a.group;
  } else if constexpr (SCORED) {
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
      const int h = head0 + 16 * cb + c;
      keep.at[cb] = h < a.group ? 16u * (g * a.group + h) : 0x7fffffffu;
    }
  }
  auto step = [&](Regs& now, Regs& ahead) -> bool {
    load(ahead);
    pages = fetch(u + 2 * W);
    const int tok0 = token0(u);
    if (!SCORED && tok0 + kUnit - 1 >= r.sinks && tok0 < r.start) {
#pragma unroll
      for (int i = 0; i < kUnit / 4; ++i) now.bmask &= r.attends(tok0 + kUnit / 4 * g + i) ? ~0u : ~(1u << i);
    }
    if constexpr (WHOLE)
      keep.unit = s_raw + u * a.group * kUnit;
    else if constexpr (SCORED)
      keep.unit = bounded_rsrc(raw + static_cast<int64_t>(u) * a.group * (4 * kUnit), 4 * kUnit * a.group);
    if constexpr (DM)
      process_unit_dm<T, false, D, false>(now, qf[0], a.scale_log2, tok0, 0, r.len - 1, -1, DmAppendRegs<D>{}, lane,
                                          s_stage + wave * D * kDmRowBytes, st[0], keep);
    else
      process_unit<T, false, kBoundedUnit, D, NCB, false, false>(now, qf, a.scale_log2, tok0, 0, r.len - 1, -1,
                                                                 AppendRegs<D>{}, c, g, st, keep);
    u += W;
    return u < u_end;
  };
  if (u < u_end)
    while (step(ra, rb) && step(rb, ra)) {
    }

  // the waves' states meet in LDS; thread -> (head, N dims)
  constexpr int N = D == 128 ? 8 : 4;
  static_assert(64 * W == 16 * (D / N), "a thread for each");
  constexpr int kSpread = acc_spread<D>();
  const int h = threadIdx.x / (D / N), d0 = (threadIdx.x % (D / N)) * N;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    if (cb > 0) __syncthreads();
    const float lt = column_sum(st[cb].l);
    if (g == 0) {
      s_m[wave][c] = st[cb].m;
      s_l[wave][c] = lt;
    }
    if constexpr (DM) {  // this lane's dims 16 n + 4 g ..
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        if (WHOLE && c >= acc_rows) break;
        *reinterpret_cast<f32x4*>(s_acc + (wave * acc_rows + c) * P + kSpread * (16 * n + 4 * g)) = st[0].acc[n];
      }
    } else {
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        if (WHOLE && c >= acc_rows) break;
        float* dst = s_acc + (wave * acc_rows + c) * P + kSpread * ((D / 4) * g + (D / 16) * rr);
        const WaveState<D>& x = st[cb];
        *reinterpret_cast<f32x4*>(dst) = f32x4{x.acc[0][rr], x.acc[1][rr], x.acc[2][rr], x.acc[3][rr]};
        if constexpr (D == 128)
          *reinterpret_cast<f32x4*>(dst + 4) = f32x4{x.acc[4][rr], x.acc[5][rr], x.acc[6][rr], x.acc[7][rr]};
      }
    }
    __syncthreads();
    const int head = head0 + 16 * cb + h;
    if (head >= a.group) continue;
    float M = -INFINITY, L = 0.f;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < W; ++x) M = fmaxf(M, s_m[x][h]);
    const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float wt = exp2_fast(s_m[x][h] - mu);
      L += wt * s_l[x][h];
      const f32x4 y = *reinterpret_cast<const f32x4*>(s_acc + (x * acc_rows + h) * P + kSpread * d0);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += wt * y[j];
      if constexpr (N == 8) {
        const f32x4 z = *reinterpret_cast<const f32x4*>(s_acc + (x * acc_rows + h) * P + d0 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[4 + j] += wt * z[j];
      }
    }
    const int qh = kvh * a.group + head;
    if (WHOLE && d0 == 0) s_z[h] = L == 0.f ? INFINITY : M + __log2f(L);
    if (WHOLE || (!SCORED && chunks == 1)) {
      const float inv = L > 0.f ? rcp_fast(L) : 0.f;
      T* dst = static_cast<T*>(a.out) + static_cast<int64_t>(b) * a.os0 + static_cast<int64_t>(qh) * a.os1 +
               static_cast<int64_t>(d0) * a.os2;
      if (a.out_rows) {
        const u32x2 lo{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
        if constexpr (N == 8)
          *reinterpret_cast<u32x4*>(dst) =
              u32x4{lo[0], lo[1], pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv)};
        else
          *reinterpret_cast<u32x2*>(dst) = lo;
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) dst[static_cast<int64_t>(j) * a.os2] = from_f32<T>(o[j] * inv);
      }
    } else {
      const int64_t at = (static_cast<int64_t>(b) * a.hq + qh) * chunks + chunk;
      float* dst = a.acc + at * D + d0;
      *reinterpret_cast<f32x4*>(dst) = f32x4{o[0], o[1], o[2], o[3]};
      if constexpr (N == 8) *reinterpret_cast<f32x4*>(dst + 4) = f32x4{o[4], o[5], o[6], o[7]};
      if (d0 == 0) a.stats[at] = float2{M, L};
    }
  }
  if constexpr (WHOLE) {
    __syncthreads();
    float* scores = a.scores + b * a.scs0 + kvh * a.scs1;
    auto add = [&](auto odd) {
      for (int t = 4 * static_cast<int>(threadIdx.x); t < r.len; t += 256 * W) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < a.group; ++x) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(s_raw + raw_at(t, x, a.group));
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] += token_weight<odd>(y[i], s_z[x]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < r.len) scores[t + i] += sum[i];
      }
    };
    if (any_nan(s_z, a.group))
      add(std::true_type{});
    else
      add(std::false_type{});
  }
}

// ============================================================== join =====
constexpr int kJoinRows = 4;       // (request, query head) rows of a join workgroup, one per wave
constexpr int kJoinTokens = 1024;  // tokens of a weights workgroup, four a thread
constexpr int kJoinHeads = 64;     // heads whose M + log2 L a weights workgroup holds at once
constexpr int kJoinAhead = 16;     // partial rows on their way at once
static_assert(kJoinAhead * kJoinRows == 64, "a wave holds the statistics of the chunks that the waves read at once");
// Weights workgroups a CU, which take a pair's spans of kJoinTokens in turn: all
// resident at once beside the rows'.  16 rows of 128 .. 32768 tokens, Hq 14, Hkv 2,
// D 64: the join 10.8, 8.0, 7.5, 9.7 us with 1 .. 4, one for every span 8.8.  Whole calls
// with 1 .. 4, rows of 32 .. 8192 tokens, Hq 32, Hkv 8, D 128: 16 rows 34.4, 32.5, 32.5,
// 32.9, 32 rows 58.1, 53.8, 52.9, 52.5; few long rows, equal rows and 71 heads a KV head
// within 1.5 % with any.
constexpr int kJoinSlots = 3;

// What is read after the first loads have gone out.
struct JoinArgs {
  void* out;
  int64_t os0, os1, os2;
  float* scores;
  int64_t scs0, scs1;
  int32_t rows, cap, window, sinks, chunk_tiles, units;
};

// Over the wave, every lane receiving the result: rotations within each 16-lane
// row, then across the rows.
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float join_max(float x) {
  x = fmaxf(x, dpp_f32<0x128>(x));
  x = fmaxf(x, dpp_f32<0x124>(x));
  x = fmaxf(x, dpp_f32<0x122>(x));
  x = fmaxf(x, dpp_f32<0x121>(x));
  return column_max(x);
}
__device__ __forceinline__ float join_sum(float x) {
  x += dpp_f32<0x128>(x);
  x += dpp_f32<0x124>(x);
  x += dpp_f32<0x122>(x);
  x += dpp_f32<0x121>(x);
  return column_sum(x);
}

// A row's M and L, of which the lanes hold the first 128 chunks' (M, L) in `x` and `y`.
__device__ __forceinline__ float2 join_stats(float2 x, float2 y, const float2* st, int live, int lane) {
  float m = lane < live ? x.x : -INFINITY, l = lane < live ? x.y : 0.f;
  auto add = [&](float2 z) {
    const float n = fmaxf(m, z.x), u = n == -INFINITY ? 0.f : n;
    l = l * exp2_fast(m - u) + z.y * exp2_fast(z.x - u);
    m = n;
  };
  if (lane + 64 < live) add(y);
  for (int c = lane + 128; c < live; c += 64) add(st[c]);
  const float M = join_max(m), u = M == -INFINITY ? 0.f : M;
  return float2{M, join_sum(l * exp2_fast(m - u))};
}

// Workgroups [0, row_blocks): out rows, one wave each, or where there are more chunks
// than a wave reads at once, four.  The rest (scored): the weights of a pair's tokens,
// four a thread.  Short and bound by its dependent
// loads: the leading arguments are preloaded into SGPRs, and the first partials,
// statistics and scores are asked for before the row's length says how many of
// them there are (a chunk without tokens holds what an earlier call left: it is
// selected away).  RAW: heads' scores on their way at once, 4 for groups of up to
// 4, else 8 (0: not scored).
template <typename T, int D, int RAW>
__global__ __launch_bounds__(256) void bounded_join_kernel(const float* acc_, const float2* stats, const void* sl,
                                                           const float* raw_, int32_t sls, int32_t hkv, int32_t group,
                                                           int32_t chunks_i64, int32_t row_blocks,
                                                           int32_t spans, JoinArgs a) {
  constexpr int E = D / 64;  // dims a lane, neighbours
  const int hq = hkv * group, chunks = chunks_i64 >> 1, sl_i64 = chunks_i64 & 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto plan = [&](int32_t len) {
    const BoundedRow r = bounded_row(len, a.cap, a.window, a.sinks);
    return (r.tiles + a.chunk_tiles - 1) / a.chunk_tiles;
  };
  if (static_cast<int>(blockIdx.x) < row_blocks) {
    // more chunks than a wave reads at once: the waves share a row
    const bool shared = chunks > kJoinAhead;
    const int row = shared ? blockIdx.x : blockIdx.x * kJoinRows + wave;
    const int start = shared ? kJoinAhead * wave : 0;
    if (row >= a.rows) return;
    const int b = row / hq, qh = row - b * hq;
    const int32_t len = load_index_uniform(sl, static_cast<int64_t>(b) * sls, sl_i64);
    const float2* st = stats + static_cast<int64_t>(row) * chunks;
    const float* acc = acc_ + static_cast<int64_t>(row) * chunks * D + E * lane;
    const float2 first = st[min(lane, chunks - 1)];
    float2 second = first;
    if (chunks > 64) second = st[min(lane + 64, chunks - 1)];
    float x[kJoinAhead][E];
    auto load = [&](int c0) {
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const float* from = acc + static_cast<int64_t>(min(c0 + j, chunks - 1)) * D;
        if constexpr (E == 2) {
          const float2 y = *reinterpret_cast<const float2*>(from);
          x[j][0] = y.x;
          x[j][1] = y.y;
        } else {
          x[j][0] = *from;
        }
      }
    };
    load(start);
    const int live = plan(len);
    const float2 ml = join_stats(first, second, st, live, lane);
    const float u = ml.x == -INFINITY ? 0.f : ml.x;
    float o[E] = {};
    float2 part = first;
    for (int c0 = start; c0 < live; c0 += kJoinAhead * kJoinRows) {  // (once, where a wave has a row)
      if (c0 > start) {
        part = st[min((c0 & ~63) + lane, chunks - 1)];
        load(c0);
      }
      const float wl = exp2_fast(part.x - u);  // of chunk (c0 & ~63) + lane
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const float wt = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wl), (c0 & 63) + j));
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += c0 + j < live ? wt * x[j][e] : 0.f;
      }
    }
    if (shared) {
      __shared__ float s_o[kJoinRows][D];
#pragma unroll
      for (int e = 0; e < E; ++e) s_o[wave][E * lane + e] = o[e];
      __syncthreads();
      if (wave > 0) return;
#pragma unroll
      for (int e = 0; e < E; ++e)
        for (int w = 1; w < kJoinRows; ++w) o[e] += s_o[w][E * lane + e];
    }
    const float inv = ml.y > 0.f ? 1.f / ml.y : 0.f;
    T* dst = static_cast<T*>(a.out) + b * a.os0 + qh * a.os1 + E * lane * a.os2;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e * a.os2] = from_f32<T>(o[e] * inv);
    return;
  }
  if constexpr (RAW > 0) {
    __shared__ float s_z[kJoinHeads];  // M + log2 L of each head
    const int at = blockIdx.x - row_blocks;
    const int pair = at / spans, first = at - pair * spans;
    const int b = pair / hkv, kvh = pair - b * hkv;
    const int32_t len = load_index_uniform(sl, static_cast<int64_t>(b) * sls, sl_i64);
    const float2* st = stats + (static_cast<int64_t>(b) * hq + kvh * group) * chunks;
    float2 y[4][2];
    auto load_stats = [&](int h, int last) {  // of this wave's heads h, h + 4 ..
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2* from = st + static_cast<int64_t>(min(h + 4 * j, last)) * chunks;
        y[j][0] = y[j][1] = from[min(lane, chunks - 1)];
        if (chunks > 64) y[j][1] = from[min(lane + 64, chunks - 1)];
      }
    };
    load_stats(wave, min(kJoinHeads, group) - 1);
    const float* raw = raw_ + static_cast<int64_t>(pair) * a.units * group * 16;
    float* row = a.scores + b * a.scs0 + kvh * a.scs1;
    f32x4 old;
    auto load_old = [&](int span, int end) {
      const int tok = span * kJoinTokens + 4 * static_cast<int>(threadIdx.x);
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = tok + i < end ? row[tok + i] : 0.f;
    };
    load_old(first, a.cap);
    const BoundedRow r = bounded_row(len, a.cap, a.window, a.sinks);
    const int live = (r.tiles + a.chunk_tiles - 1) / a.chunk_tiles;
    for (int span = first; span * kJoinTokens < r.len; span += spans) {
      const int tok = span * kJoinTokens + 4 * static_cast<int>(threadIdx.x);
      const bool there = tok < r.len;
      f32x4 x[RAW];
      auto load = [&](int h0) {
#pragma unroll
        for (int j = 0; j < RAW; ++j)
          x[j] = there ? *reinterpret_cast<const f32x4*>(raw + raw_at(tok, min(h0 + j, group - 1), group))
                       : f32x4{0.f, 0.f, 0.f, 0.f};
      };
      load(0);
      if (span > first) load_old(span, r.len);
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      for (int h0 = 0; h0 < group; h0 += kJoinHeads) {
        const int n = min(kJoinHeads, group - h0);
        if (span == first || group > kJoinHeads) {
          if (span > first || h0 > 0) __syncthreads();
          for (int h = wave; h < n; h += 4 * 4) {  // four heads of a wave at once
            if (span > first || h0 + h > wave) load_stats(h0 + h, h0 + n - 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (h + 4 * j >= n) break;
              const float2 ml =
                  join_stats(y[j][0], y[j][1], st + static_cast<int64_t>(h0 + h + 4 * j) * chunks, live, lane);
              if (lane == 0) s_z[h + 4 * j] = ml.y == 0.f ? INFINITY : ml.x + __log2f(ml.y);
            }
          }
          __syncthreads();
        }
        auto add = [&](auto odd) {
          for (int h = 0; h < n; h += RAW) {
            if (h0 + h > 0) load(h0 + h);
#pragma unroll
            for (int j = 0; j < RAW; ++j) {
              const float z = s_z[min(h + j, n - 1)];
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[i] += h + j < n ? token_weight<odd>(x[j][i], z) : 0.f;
            }
          }
        };
        if (any_nan(s_z, n))
          add(std::true_type{});
        else
          add(std::false_type{});
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tok + i < r.len) row[tok + i] = old[i] + sum[i];
    }
  }
}

// ========================================================== host glue ====
namespace {

struct BoundedPlan {
  int64_t chunk_tiles = 1, chunks = 1, units = 0;
  int64_t acc = 0, stats = 0, raw = 0;  // floats
  int64_t floats() const { return acc + stats + raw; }
};

// Tiles of a chunk for rows of `tiles` tiles, `wgs` workgroups a chunk.  A CU's
// time is its workgroups' tiles and about two tiles more for the start and end of
// each; a second chunk costs the join, about four; every CU is taken to have as many
// workgroups as the fullest, up to three.  Of the counts within a
// sixteenth of the least cost the largest: short rows then end sooner.  Groups above 16
// heads fit twice and take the least cost (Hq 71, Hkv 1, D 64, 16 rows of 129 tiles in 5
// / 10 chunks 15.8 / 19.7; Hq 40, Hkv 2, 24 rows in 5 / 8 23 / 30).  MI355X,
// 128-dim heads, us a call at 1, 2, 3, 4, 5, 8 chunks a row, * the least cost: 129
// tiles: 32 pairs 57, 34, 26, 21, 19, 15*; 64 59, 37, 28, 25*, 33, 26; 96 62, 39, 50,
// 41, 36*, 36; 192 70, 75, 76, 65*, 67, 68; 256 79*, 83, 84, 86, 86, 90; 384 139,
// 123*, 131, 127, 132, 137.  33 tiles: 64 pairs 16.5, 14.1, 11.9, 11.0*, 12.9; 160
// 19.2, 23, 18.7*; 192 20.0*, 24, 24, 22.  129 tiles, 104 pairs in 5 / 7* 48 / 39, 152
// in 4 / 5* 61 / 53, 184 in 3 / 4* 76 / 65; in 3 where 1 is the least, 208 pairs 78 / 75
// with full rows and 44 / 54 with rows from 1 / 256 of that on.  64-dim heads have
// the same order at about 0.55 of it.  Dim-major 128-dim workgroups (67 KB of LDS) fit
// twice, not three times, and of a group's heads blocks of 16 are launched where blocks
// of 32 are counted; the counts are good for them too (128 tiles, 152, 176, 184, 192
// pairs: 55.5, 63.1, 65.5, 72.3 us, counted with two slots 55.4, 71.2, 71.0, 71.4).
constexpr int64_t kChunkStart = 2, kChunkJoin = 4;

int64_t chunk_tiles_for(int64_t wgs, int64_t tiles, int64_t cus, bool wide) {
  // (a thread's calls mostly repeat: the last answer is kept, for half a us a call)
  static thread_local int64_t last[5] = {0, 0, 0, 0, 0};
  if (last[0] == wgs && last[1] == tiles && last[2] == cus && last[4] == wide) return last[3];
  const int64_t slots = wide ? 2 : 3, near = wide ? 0 : 1;
  auto counts = [&](auto take) {
    for (int64_t n = 1; n == 1 || (n * wgs <= slots * cus && 2 * n <= tiles + 1); ++n) {
      const int64_t per = (tiles + n - 1) / n, all = (tiles + per - 1) / per * wgs;
      take(per, (all + cus - 1) / cus * (per + kChunkStart) + (n > 1 ? kChunkJoin : 0));
    }
  };
  int64_t best = tiles, least = INT64_MAX;
  counts([&](int64_t, int64_t cost) { least = cost < least ? cost : least; });
  counts([&](int64_t per, int64_t cost) { best = 16 * cost <= (16 + near) * least ? per : best; });
  last[0] = wgs;
  last[1] = tiles;
  last[2] = cus;
  last[4] = wide;
  return last[3] = best < 2 ? 2 : best;
}

// A scored row may be far shorter than its table, and batches of unequal rows come
// out even in short chunks only, the more so the fewer rows there are.  Hq 32, Hkv 8
// (* Hq 16, Hkv 2), us a call at 4, 8, 11, 16, 32 tiles a chunk: rows of 1 / 256 of
// the table to all of it: 32* pairs of 1024 tiles -, 35.1, 39.5, 45.7, 55.2; 128 of
// 256 30.3, 30.6, 33.0, 37.2, 42.1; 512 of 128 59.0, 54.9, 55.1, 58.3, 72.0.  Rows of
// half of it to all: 128 pairs of 128 tiles 50.8, 48.6, 47.5, 50.0, 59.5; 256 of 256
// 187.8, 184.1, 177.9, 177.4, 180.4.
constexpr int64_t kScoredTilesFew = 8, kScoredTilesMany = 11;

// Whole scored rows, one workgroup each, where the group and a row of a full table
// leave room in LDS: no scores or partials go through memory and nothing is joined
// (25 MB of scores among 805 MB of K/V cost the chunks a fifth of their time, mostly
// as writes).  A workgroup alone on its CU takes 0.4 us a tile, so it has to be short
// (kWholeTiles), or there is one for most of the CUs, in the last round too, and the
// caller does not say that lengths vary widely.  Us a call in chunks / whole, Hq 16, Hkv 2 (* Hq 32, Hkv 8):
//   2 pairs of 2 tiles 7.6 / 4.6, of 8 7.5 / 6.3, of 12 7.5 / 7.5; 16 of 10 8.3 / 8.2,
//     of 12 8.3 / 9.0; 64 of 10 9.1 / 8.9; 128 of 16 11.4 / 11.8;
//   192* of 32 27.0 / 20.9, of 256 174 / 143; 256* of 32 29.9 / 23.4, of 256 230 / 166,
//     rows from half of that on 177 / 147, rows spread from 1 / 256 of it on 53 / 114;
//     264* of 256 242 / 283, 184 / 161, 320* 292 / 292, 221 / 226, 384* 349 / 309,
//     267 / 252; 352* of 128 162 / 150, 126 / 135, 384* 175 / 153, 137 / 128, 512* 229 / 168,
//     178 / 143, 56 / 77.
constexpr int64_t kWholeTiles = 10;
constexpr int64_t kWholeLds = 158 << 10;

// Bytes of LDS beside the fixed ones: the waves' states and the row's scores.
int64_t whole_lds(int64_t group, int64_t tiles) {
  return 4 * group * (kWholeWaves * acc_pitch<128>() + 32 * tiles);
}

bool scored_whole(const fd_paged_decode_args& a, int64_t tiles, bool ragged, bool dm) {
  const int64_t group = a.num_q_heads / a.num_kv_heads, pairs = a.num_seqs * a.num_kv_heads;
  const int64_t stage = dm ? kWholeWaves * a.head_dim * kDmRowBytes : 0;
  if (group > 16 || whole_lds(group, tiles) + stage > kWholeLds) return false;
  const int64_t cus = device_cus();
  return tiles <= kWholeTiles || (!ragged && (pairs <= cus ? 4 * pairs >= 3 * cus : 2 * pairs >= 3 * cus));
}

// Workgroups that share a (request, KV head, chunk): query heads of the group in
// blocks of 16 or, past 16, of 32 (8 in the generic kernel).
int64_t head_blocks(const fd_paged_decode_args& a) {
  const int64_t group = a.num_q_heads / a.num_kv_heads;
  return group <= 16 ? 1 : (group + 31) / 32;
}
int64_t generic_head_blocks(const fd_paged_decode_args& a) {
  return (a.num_q_heads / a.num_kv_heads + kBoundedHeads - 1) / kBoundedHeads;
}

// Workgroups that share a pair's weights.
int64_t join_spans(const fd_paged_decode_args& a) {
  return (a.max_blocks_per_seq * a.block_size + kJoinTokens - 1) / kJoinTokens;
}

int64_t up4(int64_t x) { return (x + 3) & ~int64_t{3}; }

// fill_decode_params has checked the shapes.
BoundedPlan bounded_plan(const fd_paged_decode_args& a, int window, int sinks, bool scored) {
  BoundedPlan s;
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  const int64_t tiles = bounded_max_tiles(cap, window, sinks);
  const int64_t wgs = a.num_seqs * a.num_kv_heads * head_blocks(a);  // of one chunk a row
  int64_t per = chunk_tiles_for(wgs, tiles, device_cus(), a.num_q_heads / a.num_kv_heads > 16);
  if (scored) {
    const int64_t most = wgs < device_cus() ? kScoredTilesFew : kScoredTilesMany;
    per = per < most ? per : most;
  }
  const int64_t most = 65535 / generic_head_blocks(a);  // chunks that the grid's second dimension holds
  if (tiles > per * most) per = (tiles + most - 1) / most;
  s.chunks = (tiles + per - 1) / per;
  s.chunk_tiles = (tiles + s.chunks - 1) / s.chunks;
  s.chunks = (tiles + s.chunk_tiles - 1) / s.chunk_tiles;
  // (an odd count: pairs a power of two apart would meet in the same memory channels,
  // the join of 32 x 6144 tokens, Hq 32, Hkv 8, 12.9 -> 11.9 us)
  s.units = 2 * ((cap + 31) / 32) + 1;
  const int64_t rows = a.num_seqs * a.num_q_heads;
  if (s.chunks > 1 || scored) {
    s.acc = rows * s.chunks * a.head_dim;
    s.stats = up4(2 * rows * s.chunks);
  }
  if (scored) s.raw = rows * s.units * 16;
  return s;
}

bool fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

// The MFMA kernel's calls: the row kernel's (fast_path_ok), with 32-bit strides, and
// their like of dim-major caches (a block's dims within 32-bit byte offsets).
bool bounded_small(const fd_paged_decode_args& a) {
  for (int64_t x : {a.q_stride[0], a.q_stride[1], a.out_stride[0], a.out_stride[1], a.out_stride[2], a.seq_lens_stride,
                    a.num_blocks, a.num_q_heads})
    if (!fits32(x)) return false;
  return a.num_seqs <= 65535 && a.num_kv_heads <= 65535;  // the grid's second and third dimension
}

bool bounded_fast(const fd_paged_decode_args& a) {
  if (!fast_path_ok(a, a.num_q_heads / a.num_kv_heads)) return false;
  for (const int64_t* st : {a.k_stride, a.v_stride})
    for (int i = 0; i < 3; ++i)
      if (!fits32(st[i])) return false;
  return bounded_small(a);
}

bool bounded_dm(const fd_paged_decode_args& a) {
  if (a.num_q_heads / a.num_kv_heads > 256 || a.q_stride[2] != 1) return false;
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15u)
    return false;
  if (a.q_stride[0] % 8 || a.q_stride[1] % 8) return false;
  for (const int64_t* st : {a.k_stride, a.v_stride}) {
    if (st[2] != 1 || st[0] % 8 || st[1] % 8 || st[3] % 8) return false;
    if (!fits32(st[0]) || !fits32(st[1]) || st[3] < 0 || 2 * (a.head_dim * st[3] + a.block_size) > INT32_MAX) return false;
  }
  for (int64_t t : {a.block_tables_stride[0], a.block_tables_stride[1], a.max_blocks_per_seq})
    if (!fits32(t)) return false;
  return bounded_small(a);
}

BoundedArgs bounded_args(const fd_paged_decode_args& a, const DecodeParams& p, const BoundedParams& w, bool dm) {
  auto i32 = [](int64_t x) { return static_cast<int32_t>(x); };
  BoundedArgs e{};
  e.q = a.q;
  e.k = a.k_cache;
  e.v = a.v_cache;
  e.bt = a.block_tables;
  e.sl = a.seq_lens;
  e.out = a.out;
  e.acc = w.acc;
  e.stats = w.stats;
  e.raw = w.raw;
  e.scores = w.scores;
  e.scs0 = w.scs0;
  e.scs1 = w.scs1;
  e.qs0 = i32(a.q_stride[0]);
  e.qs1 = i32(a.q_stride[1]);
  e.ks0 = i32(a.k_stride[0]);
  e.ks1 = i32(a.k_stride[1]);
  e.ks2 = i32(a.k_stride[dm ? 3 : 2]);
  e.vs0 = i32(a.v_stride[0]);
  e.vs1 = i32(a.v_stride[1]);
  e.vs2 = i32(a.v_stride[dm ? 3 : 2]);
  e.bts0 = i32(a.block_tables_stride[0]);
  e.bts1 = i32(a.block_tables_stride[1]);
  e.sls = i32(a.seq_lens_stride);
  e.os0 = i32(a.out_stride[0]);
  e.os1 = i32(a.out_stride[1]);
  e.os2 = i32(a.out_stride[2]);
  e.out_rows = a.out_stride[2] == 1 && a.out_stride[0] % 8 == 0 && a.out_stride[1] % 8 == 0 &&
               (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
  e.i64 = (p.sl_i64 ? 1 : 0) | (p.bt_i64 ? 2 : 0);
  e.num_blocks = i32(a.num_blocks);
  e.hkv = p.hkv;
  e.hq = p.hq;
  e.group = p.group;
  e.width = i32(a.max_blocks_per_seq);
  e.cap = i32(a.max_blocks_per_seq * a.block_size);
  e.window = w.window;
  e.sinks = w.sinks;
  e.chunk_tiles = w.chunk_tiles;
  e.chunks = w.chunks;
  e.units = w.units;
  e.scale_log2 = p.scale_log2;
  return e;
}

template <typename T, int D, int MODE, int W, int NCB, bool DM = false>
void launch_bounded_mfma(const fd_paged_decode_args& a, const BoundedArgs& e, hipStream_t stream) {
  const int64_t blocks = DM ? (e.group + 15) / 16 : head_blocks(a);
  const bool rounds = a.num_seqs * a.num_kv_heads * e.chunks * blocks > device_cus();
  const dim3 grid(static_cast<unsigned>((e.chunks | (rounds ? 1 : 0)) * blocks),
                  static_cast<unsigned>(a.num_kv_heads), static_cast<unsigned>(a.num_seqs));
  auto go = [&](auto kernel) {
    const uint32_t lds = MODE == kScoredWhole ? static_cast<uint32_t>(whole_lds(e.group, e.chunk_tiles)) : 0u;
    dispatch_lds(kernel, grid, dim3(64 * W), lds, stream, a.timing_events[0], a.timing_events[1], e.sl, e.bt, e.sls,
                 e.bts0, e.bts1, e.hkv, e.chunks, e.chunk_tiles, e.cap, e.window, e.sinks, e.i64, e);
  };
  const bool nt = a.kv_reuse == 0;
  switch (a.block_size) {
    case 8:
      nt ? go(bounded_mfma_kernel<T, 8, D, NCB, MODE, W, true, DM>)
         : go(bounded_mfma_kernel<T, 8, D, NCB, MODE, W, false, DM>);
      break;
    case 16:
      nt ? go(bounded_mfma_kernel<T, 16, D, NCB, MODE, W, true, DM>)
         : go(bounded_mfma_kernel<T, 16, D, NCB, MODE, W, false, DM>);
      break;
    default:
      nt ? go(bounded_mfma_kernel<T, 32, D, NCB, MODE, W, true, DM>)
         : go(bounded_mfma_kernel<T, 32, D, NCB, MODE, W, false, DM>);
      break;
  }
}

template <typename T, int D, bool SCORED>
int launch_bounded(const fd_paged_decode_args& a, const DecodeParams& p, BoundedParams w, const char* fn,
                   hipStream_t stream) {
  const int64_t pairs = a.num_seqs * a.num_kv_heads;
  const int64_t tiles = bounded_max_tiles(a.max_blocks_per_seq * a.block_size, w.window, w.sinks);
  constexpr int kMode = SCORED ? kScored : kWindow;
  const bool fast = bounded_fast(a), dm = !fast && bounded_dm(a);
  const bool whole = SCORED && (fast || dm) && scored_whole(a, tiles, w.ragged, dm);
  const bool joins = !whole && (SCORED || w.chunks > 1);
  const int64_t rows = a.num_seqs * a.num_q_heads;
  const int64_t row_blocks = w.chunks > kJoinAhead ? rows : (rows + kJoinRows - 1) / kJoinRows;
  // weights workgroups of a pair: kJoinSlots a CU over all pairs
  const int64_t slots = (kJoinSlots * device_cus() + pairs - 1) / pairs;
  const int64_t spans = !SCORED ? 0 : join_spans(a) < slots ? join_spans(a) : slots;
  if ((!fast && !dm && !grid_fits(pairs, 64)) || (joins && !grid_fits(row_blocks + pairs * spans, 256)))
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  if (fast || dm) {
    if (whole) {
      w.chunks = 1;
      w.chunk_tiles = static_cast<int>(tiles);
    }
    const BoundedArgs e = bounded_args(a, p, w, dm);
    if (whole)
      dm ? launch_bounded_mfma<T, D, kScoredWhole, kWholeWaves, 1, true>(a, e, stream)
         : launch_bounded_mfma<T, D, kScoredWhole, kWholeWaves, 1>(a, e, stream);
    else if (dm)
      launch_bounded_mfma<T, D, kMode, kBoundedWaves, 1, true>(a, e, stream);
    else if (p.group > 16)
      launch_bounded_mfma<T, D, kMode, kBoundedWaves, 2>(a, e, stream);
    else
      launch_bounded_mfma<T, D, kMode, kBoundedWaves, 1>(a, e, stream);
  } else {
    const int hg = static_cast<int>(generic_head_blocks(a));
    const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(hg * w.chunks));
    dispatch(bounded_generic_kernel<T, D, SCORED>, grid, dim3(64), stream, a.timing_events[0], a.timing_events[1], p, w,
             hg);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "bounded decode launch failed: %s", hipGetErrorString(e));
  if (!joins) return FD_OK;
  JoinArgs j{};
  j.out = p.out;
  j.os0 = p.os0;
  j.os1 = p.os1;
  j.os2 = p.os2;
  j.scores = w.scores;
  j.scs0 = w.scs0;
  j.scs1 = w.scs1;
  j.rows = static_cast<int32_t>(rows);
  j.cap = static_cast<int32_t>(a.max_blocks_per_seq * a.block_size);
  j.window = w.window;
  j.sinks = w.sinks;
  j.chunk_tiles = w.chunk_tiles;
  j.units = w.units;
  auto join = [&](auto kernel) {
    dispatch(kernel, dim3(static_cast<unsigned>(row_blocks + pairs * spans)), dim3(256), stream, a.timing_events[2],
             a.timing_events[3], static_cast<const float*>(w.acc), static_cast<const float2*>(w.stats), p.sl,
             static_cast<const float*>(w.raw), static_cast<int32_t>(p.sls), p.hkv, p.group, 2 * w.chunks + (p.sl_i64 ? 1 : 0),
             static_cast<int32_t>(row_blocks), static_cast<int32_t>(spans), j);
  };
  if constexpr (SCORED)
    p.group <= 4 ? join(bounded_join_kernel<T, D, 4>) : join(bounded_join_kernel<T, D, 8>);
  else
    join(bounded_join_kernel<T, D, 0>);
  e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "bounded decode join launch failed: %s", hipGetErrorString(e));
  return FD_OK;
}

// What both entry points ask of the decode arguments beside fill_decode_params.
int bounded_check(const fd_paged_decode_args* args, const char* fn, DecodeParams& p) {
  const int rc = fill_decode_params(args, fn, p);
  if (rc != FD_OK) return rc;
  const fd_paged_decode_args& a = *args;
  if (a.num_splits != 1 || a.split_counters || a.balance_target)
    return set_error(FD_E_INVALID, "%s: takes num_splits 1 and no split workspace, counters or balance_target", fn);
  if (a.append_k || a.rotary_dim)
    return set_error(FD_E_UNSUPPORTED, "%s: no fused append or RoPE (append first)", fn);
  if (a.seq_lens_stride < 0 || a.seq_lens_stride > INT32_MAX)
    return set_error(FD_E_UNSUPPORTED, "%s: seq_lens stride does not fit 32 bits", fn);
  if (a.max_blocks_per_seq > INT32_MAX || a.max_blocks_per_seq * a.block_size > INT32_MAX - 4096)
    return set_error(FD_E_UNSUPPORTED, "%s: block tables hold 2^31 tokens or more", fn);
  // (the plan divides the grid's second dimension by them)
  if (generic_head_blocks(a) > 65535) return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

int check_window(const fd_window_args* win, const char* fn) {
  if (win == nullptr) return set_error(FD_E_INVALID, "%s: window is NULL", fn);
  if (win->struct_size != sizeof(fd_window_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, win->struct_size,
                     sizeof(fd_window_args));
  if (win->window < 1 || win->sink_tokens < 0)
    return set_error(FD_E_INVALID, "%s: window must be positive and sink_tokens non-negative", fn);
  return FD_OK;
}

int check_scores(const fd_paged_decode_args& a, const fd_score_args* sc, const char* fn) {
  if (sc == nullptr) return set_error(FD_E_INVALID, "%s: scores is NULL", fn);
  if (sc->struct_size != sizeof(fd_score_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, sc->struct_size,
                     sizeof(fd_score_args));
  if (sc->scores == nullptr) return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (sc->ragged != 0 && sc->ragged != 1) return set_error(FD_E_INVALID, "%s: ragged must be 0 or 1", fn);
  if (sc->tokens < a.max_blocks_per_seq * a.block_size)
    return set_error(FD_E_INVALID, "%s: scores must hold every token of a block-table row", fn);
  return FD_OK;
}

// The launch grids are 32-bit, and so are the indices in them.
int check_grid(const fd_paged_decode_args& a, const BoundedPlan& s, bool scored, const char* fn) {
  const int64_t pairs = a.num_seqs * a.num_kv_heads;
  const int64_t spans = scored ? join_spans(a) : 0;
  if (generic_head_blocks(a) * s.chunks > 65535 || pairs > INT32_MAX ||
      pairs * head_blocks(a) * (s.chunks + 1) > INT32_MAX || a.num_seqs * a.num_q_heads + pairs * spans > INT32_MAX)
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

template <bool SCORED>
int run_bounded(const fd_paged_decode_args& a, const DecodeParams& p, BoundedParams w, const BoundedPlan& s,
                float* workspace, int64_t floats, const char* fn, hipStream_t stream) {
  if (s.floats() > 0 &&
      (workspace == nullptr || floats < s.floats() || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return set_error(FD_E_INVALID, "%s: needs a 16-byte aligned workspace of %lld floats", fn,
                     static_cast<long long>(s.floats()));
  w.chunk_tiles = static_cast<int>(s.chunk_tiles);
  w.chunks = static_cast<int>(s.chunks);
  w.units = static_cast<int>(s.units);
  w.acc = workspace;
  w.stats = reinterpret_cast<float2*>(workspace + s.acc);
  w.raw = workspace + s.acc + s.stats;
  const bool bf = a.dtype == FD_DTYPE_BF16;
  if (a.head_dim == 64)
    return bf ? launch_bounded<__bf16, 64, SCORED>(a, p, w, fn, stream)
              : launch_bounded<_Float16, 64, SCORED>(a, p, w, fn, stream);
  return bf ? launch_bounded<__bf16, 128, SCORED>(a, p, w, fn, stream)
            : launch_bounded<_Float16, 128, SCORED>(a, p, w, fn, stream);
}

// Windows and sink counts past the longest row mean all of it, the largest numbers too:
// everything that reckons with them takes them cut to 32 bits.
int clamp32(int64_t x) { return static_cast<int>(x < INT32_MAX ? x : INT32_MAX); }

}  // namespace

int join_rows(const RowJoin& r, bool bf16, int head_dim, const char* fn, hipStream_t stream) {
  const int64_t blocks = r.chunks > kJoinAhead ? r.rows : (r.rows + kJoinRows - 1) / kJoinRows;
  if (!grid_fits(blocks, 256)) return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  JoinArgs j{};
  j.out = r.out;
  j.os0 = r.out_stride[0];
  j.os1 = r.out_stride[1];
  j.os2 = r.out_stride[2];
  j.rows = static_cast<int32_t>(r.rows);
  j.cap = r.cap;
  j.window = INT32_MAX;
  j.chunk_tiles = r.chunk_tiles;
  auto join = [&](auto kernel) {
    dispatch(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), stream, nullptr, nullptr, r.acc, r.stats, r.seq_lens,
             static_cast<const float*>(nullptr), static_cast<int32_t>(r.seq_lens_stride), r.hkv, r.group,
             2 * r.chunks + (r.seq_lens_i64 ? 1 : 0), static_cast<int32_t>(blocks), 0, j);
  };
  if (head_dim == 64)
    bf16 ? join(bounded_join_kernel<__bf16, 64, 0>) : join(bounded_join_kernel<_Float16, 64, 0>);
  else
    bf16 ? join(bounded_join_kernel<__bf16, 128, 0>) : join(bounded_join_kernel<_Float16, 128, 0>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: join launch failed: %s", fn, hipGetErrorString(e));
  return FD_OK;
}

}  // namespace fd

using namespace fd;

extern "C" int fd_paged_decode_window_floats(const fd_paged_decode_args* args, const fd_window_args* window,
                                             int64_t* floats) {
  static const char* fn = "fd_paged_decode_window_floats";
  DecodeParams p;
  int rc = bounded_check(args, fn, p);
  if (rc == FD_OK) rc = check_window(window, fn);
  if (rc != FD_OK) return rc;
  if (floats == nullptr) return set_error(FD_E_INVALID, "%s: floats is NULL", fn);
  *floats = bounded_plan(*args, clamp32(window->window), clamp32(window->sink_tokens), false).floats();
  return FD_OK;
}

extern "C" int fd_paged_decode_window(const fd_paged_decode_args* args, const fd_window_args* window, float* workspace,
                                      int64_t floats, fd_stream_t stream) {
  clear_launch_record();
  static const char* fn = "fd_paged_decode_window";
  DecodeParams p;
  int rc = bounded_check(args, fn, p);
  if (rc == FD_OK) rc = check_window(window, fn);
  if (rc != FD_OK) return rc;
  BoundedParams w{};
  w.window = clamp32(window->window);
  w.sinks = clamp32(window->sink_tokens);
  const BoundedPlan s = bounded_plan(*args, w.window, w.sinks, false);
  rc = check_grid(*args, s, false, fn);
  if (rc != FD_OK) return rc;
  return run_bounded<false>(*args, p, w, s, workspace, floats, fn, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int fd_paged_decode_scored_floats(const fd_paged_decode_args* args, int64_t* floats) {
  static const char* fn = "fd_paged_decode_scored_floats";
  DecodeParams p;
  const int rc = bounded_check(args, fn, p);
  if (rc != FD_OK) return rc;
  if (floats == nullptr) return set_error(FD_E_INVALID, "%s: floats is NULL", fn);
  *floats = bounded_plan(*args, INT32_MAX, 0, true).floats();
  return FD_OK;
}

extern "C" int fd_paged_decode_scored(const fd_paged_decode_args* args, const fd_score_args* scores, float* workspace,
                                      int64_t floats, fd_stream_t stream) {
  clear_launch_record();
  static const char* fn = "fd_paged_decode_scored";
  DecodeParams p;
  int rc = bounded_check(args, fn, p);
  if (rc == FD_OK) rc = check_scores(*args, scores, fn);
  if (rc != FD_OK) return rc;
  const BoundedPlan s = bounded_plan(*args, INT32_MAX, 0, true);
  rc = check_grid(*args, s, true, fn);
  if (rc != FD_OK) return rc;
  BoundedParams w{};
  w.window = INT32_MAX;
  w.sinks = 0;
  w.scores = scores->scores;
  w.ragged = scores->ragged != 0;
  w.scs0 = scores->stride[0];
  w.scs1 = scores->stride[1];
  return run_bounded<true>(*args, p, w, s, workspace, floats, fn, reinterpret_cast<hipStream_t>(stream));
}
