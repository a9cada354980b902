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
// second launch forms sum_h 2^(x_h - M_h - log2 L_h).
#include "bounded_row.h"
#include "decode_host.h"

namespace fd {

struct BoundedParams {
  int window, sinks;
  int chunk_tiles, chunks;  // tiles of a chunk; chunks of a row at most
  int units;                // 16-token units of a full table row
  float* acc;               // [row, chunk, D] (row: request, query head)
  float2* stats;            // [row, chunk] (M, L)
  float* raw;               // [pair, unit, head of the group, 16] x of every token, scored only
  float* scores;            // [request, KV head, token], scored only
  int64_t scs0, scs1;
};

__device__ __forceinline__ BoundedRow bounded_row_of(const DecodeParams& p, const BoundedParams& w, int b) {
  const int cap = static_cast<int>(p.max_blocks_per_seq * p.block_size);
  return bounded_row(load_index(p.sl, b * p.sls, p.sl_i64), cap, w.window, w.sinks);
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
  const int chunk = blockIdx.y;
  const int hg = blockIdx.x % head_groups;
  const int pair = blockIdx.x / head_groups;
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
        w.raw[((static_cast<int64_t>(pair) * w.units + tok / 16) * p.group + h0 + j) * 16 + tok % 16] = s;
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

// ============================================================== join =====
constexpr int kJoinRows = 4;      // (request, query head) rows of a join workgroup, one per wave
constexpr int kJoinTokens = 1024; // tokens of a weights workgroup
constexpr int kJoinHeads = 64;    // heads whose M + log2 L a weights workgroup holds at once

__device__ __forceinline__ float wave_max_f(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, shfl_xor_f32(x, o));
  return x;
}
__device__ __forceinline__ float wave_sum_f(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += shfl_xor_f32(x, o);
  return x;
}

// M and L of a row from its chunks' statistics, in every lane.
__device__ __forceinline__ float2 join_stats(const float2* st, int chunks, int lane) {
  float m = -INFINITY, l = 0.f;
  for (int c = lane; c < chunks; c += 64) {
    const float2 x = st[c];
    const float n = fmaxf(m, x.x);
    const float u = n == -INFINITY ? 0.f : n;
    l = l * exp2_fast(m - u) + x.y * exp2_fast(x.x - u);
    m = n;
  }
  const float M = wave_max_f(m);
  const float u = M == -INFINITY ? 0.f : M;
  return float2{M, wave_sum_f(l * exp2_fast(m - u))};
}

// Workgroups [0, row_blocks): out rows.  The rest (scored): a pair's weights,
// kJoinTokens tokens each.
template <typename T, int D, bool SCORED>
__global__ __launch_bounds__(256) void bounded_join_kernel(DecodeParams p, BoundedParams w, int row_blocks, int spans) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  if (static_cast<int>(blockIdx.x) < row_blocks) {
    const int row = blockIdx.x * kJoinRows + wave;
    if (row >= p.num_seqs * p.hq) return;
    const int b = row / p.hq, qh = row % p.hq;
    const BoundedRow r = bounded_row_of(p, w, b);
    const int chunks = (r.tiles + w.chunk_tiles - 1) / w.chunk_tiles;
    const float2* st = w.stats + static_cast<int64_t>(row) * w.chunks;
    const float* acc = w.acc + static_cast<int64_t>(row) * w.chunks * D;
    const float2 ml = join_stats(st, chunks, lane);
    const float u = ml.x == -INFINITY ? 0.f : ml.x;
    float o[D / 64];
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
    for (int c = 0; c < chunks; ++c) {
      const float wt = exp2_fast(st[c].x - u);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[e] += wt * acc[static_cast<int64_t>(c) * D + lane + 64 * e];
    }
    const float inv = ml.y > 0.f ? 1.f / ml.y : 0.f;
    T* dst = static_cast<T*>(p.out) + b * p.os0 + qh * p.os1;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) dst[(lane + 64 * e) * p.os2] = from_f32<T>(o[e] * inv);
    return;
  }
  if constexpr (SCORED) {
    __shared__ float s_z[kJoinHeads];  // M + log2 L of each head
    const int at = blockIdx.x - row_blocks;
    const int pair = at / spans, span = at % spans;
    const int b = pair / p.hkv, kvh = pair % p.hkv;
    const BoundedRow r = bounded_row_of(p, w, b);
    const int chunks = (r.tiles + w.chunk_tiles - 1) / w.chunk_tiles;
    if (span * kJoinTokens >= r.len) return;
    float sum[kJoinTokens / 256] = {};
    for (int h0 = 0; h0 < p.group; h0 += kJoinHeads) {
      const int n = min(kJoinHeads, p.group - h0);
      __syncthreads();
      for (int h = wave; h < n; h += 4) {
        const int64_t row = static_cast<int64_t>(b) * p.hq + kvh * p.group + h0 + h;
        const float2 ml = join_stats(w.stats + row * w.chunks, chunks, lane);
        // a row without a token: every weight 2^(-inf - inf) = 0
        if (lane == 0) s_z[h] = ml.y > 0.f ? ml.x + __log2f(ml.y) : INFINITY;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kJoinTokens / 256; ++i) {
        const int tok = span * kJoinTokens + 256 * i + threadIdx.x;
        if (tok >= r.len) continue;
        const float* x = w.raw + ((static_cast<int64_t>(pair) * w.units + tok / 16) * p.group + h0) * 16 + tok % 16;
        for (int h = 0; h < n; ++h) sum[i] += exp2_fast(x[16 * h] - s_z[h]);
      }
    }
#pragma unroll
    for (int i = 0; i < kJoinTokens / 256; ++i) {
      const int tok = span * kJoinTokens + 256 * i + threadIdx.x;
      if (tok < r.len) w.scores[b * w.scs0 + kvh * w.scs1 + tok] += sum[i];
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

int64_t up4(int64_t x) { return (x + 3) & ~int64_t{3}; }

// fill_decode_params has checked the shapes.
BoundedPlan bounded_plan(const fd_paged_decode_args& a, int64_t window, int64_t sinks, bool scored) {
  BoundedPlan s;
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  const int64_t tiles = bounded_max_tiles(cap, window, sinks);
  const int64_t group = a.num_q_heads / a.num_kv_heads;
  const int64_t wgs = a.num_seqs * a.num_kv_heads * ((group + kBoundedHeads - 1) / kBoundedHeads);
  // about eight waves a CU, at least two tiles and at most 32 each
  const int64_t want = (8 * device_cus() + wgs - 1) / wgs;
  s.chunk_tiles = (tiles + want - 1) / want;
  s.chunk_tiles = s.chunk_tiles < 2 ? 2 : (s.chunk_tiles > 32 ? 32 : s.chunk_tiles);
  if (tiles > 65535 * s.chunk_tiles) s.chunk_tiles = (tiles + 65534) / 65535;  // the grid's second dimension
  s.chunks = (tiles + s.chunk_tiles - 1) / s.chunk_tiles;
  s.units = 2 * ((cap + 31) / 32);
  const int64_t rows = a.num_seqs * a.num_q_heads;
  if (s.chunks > 1 || scored) {
    s.acc = rows * s.chunks * a.head_dim;
    s.stats = up4(2 * rows * s.chunks);
  }
  if (scored) s.raw = rows * s.units * 16;
  return s;
}

template <typename T, int D, bool SCORED>
int launch_bounded(const fd_paged_decode_args& a, const DecodeParams& p, const BoundedParams& w, hipStream_t stream) {
  const int64_t pairs = a.num_seqs * a.num_kv_heads;
  const int hg = (p.group + kBoundedHeads - 1) / kBoundedHeads;
  const dim3 grid(static_cast<unsigned>(pairs * hg), static_cast<unsigned>(w.chunks));
  dispatch(bounded_generic_kernel<T, D, SCORED>, grid, dim3(64), stream, a.timing_events[0], a.timing_events[1], p, w,
           hg);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "bounded decode launch failed: %s", hipGetErrorString(e));
  if (!SCORED && w.chunks == 1) return FD_OK;
  const int64_t rows = a.num_seqs * a.num_q_heads, row_blocks = (rows + kJoinRows - 1) / kJoinRows;
  const int64_t spans = SCORED ? (16 * static_cast<int64_t>(w.units) + kJoinTokens - 1) / kJoinTokens : 0;
  dispatch(bounded_join_kernel<T, D, SCORED>, dim3(static_cast<unsigned>(row_blocks + pairs * spans)), dim3(256),
           stream, a.timing_events[2], a.timing_events[3], p, w, static_cast<int>(row_blocks), static_cast<int>(spans));
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
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  if (cap > INT32_MAX - 64) return set_error(FD_E_UNSUPPORTED, "%s: block tables hold 2^31 tokens or more", fn);
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
  if (sc->tokens < a.max_blocks_per_seq * a.block_size)
    return set_error(FD_E_INVALID, "%s: scores must hold every token of a block-table row", fn);
  return FD_OK;
}

// The launch grids are 32-bit, and so are the indices in them.
int check_grid(const fd_paged_decode_args& a, const BoundedPlan& s, bool scored, const char* fn) {
  const int64_t pairs = a.num_seqs * a.num_kv_heads, group = a.num_q_heads / a.num_kv_heads;
  const int64_t spans = scored ? (16 * s.units + kJoinTokens - 1) / kJoinTokens : 0;
  if (pairs * ((group + kBoundedHeads - 1) / kBoundedHeads) * s.chunks > INT32_MAX ||
      a.num_seqs * a.num_q_heads + pairs * spans > INT32_MAX)
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
    return bf ? launch_bounded<__bf16, 64, SCORED>(a, p, w, stream)
              : launch_bounded<_Float16, 64, SCORED>(a, p, w, stream);
  return bf ? launch_bounded<__bf16, 128, SCORED>(a, p, w, stream)
            : launch_bounded<_Float16, 128, SCORED>(a, p, w, stream);
}

int clamp32(int64_t x) { return static_cast<int>(x < INT32_MAX ? x : INT32_MAX); }

}  // namespace
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
  *floats = bounded_plan(*args, window->window, window->sink_tokens, false).floats();
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
  const BoundedPlan s = bounded_plan(*args, window->window, window->sink_tokens, false);
  rc = check_grid(*args, s, false, fn);
  if (rc != FD_OK) return rc;
  BoundedParams w{};
  w.window = clamp32(window->window);
  w.sinks = clamp32(window->sink_tokens);
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
  w.scs0 = scores->stride[0];
  w.scs1 = scores->stride[1];
  return run_bounded<true>(*args, p, w, s, workspace, floats, fn, reinterpret_cast<hipStream_t>(stream));
}
