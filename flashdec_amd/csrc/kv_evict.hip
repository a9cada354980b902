// Eviction from a paged K/V cache by accumulated attention weight, for gfx950.
//
// A row of len > keep tokens keeps its first `sinks`, its last `recent` and, of
// the tokens between, the keep - sinks - recent of highest score, in their order:
//   kept = sort(sinks u recent u top(score)),  K'[j] = K[kept[j]], V', score' alike.
// Ties go to the lower index; NaN ranks below every number and -0 equals 0.
//
// kept[j] >= j, so a row is compacted in place from the front: once the sources
// of entries [j0, j1) have been read, nothing that is still to be read lies in
// front of j1.  Tokens do not mix their dimensions, heads or tensors, so each
// (request, KV head, tensor) is a stream of its own with one workgroup.
#include "decode_host.h"

namespace fd {

struct EvictParams {
  void* k;
  int64_t ks0, ks1, ks2, ks3;
  void* v;
  int64_t vs0, vs1, vs2, vs3;
  const void* bt;
  int64_t bts0, bts1;
  const void* sl;
  int64_t sls;
  const float* scores;
  int64_t scs0, scs1;
  float* new_scores;
  int64_t nss0, nss1;
  int32_t* kept;  // [request, KV head, keep]
  void* new_lens;
  int64_t nls;
  int bt_i64, sl_i64;
  int hkv, head_dim, block_size, cap;
  int keep, sinks, recent;
  int64_t num_blocks;
};

__device__ __forceinline__ int evict_len(const EvictParams& p, int b) {
  const int n = load_index(p.sl, b * p.sls, p.sl_i64);
  return n < 0 ? 0 : (n < p.cap ? n : p.cap);
}

// Order of the scores as unsigned integers: NaN 0, then -inf .. +inf, the two
// zeros alike.
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// ============================================================ select =====
constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

// One workgroup per (request, KV head).  The threshold is found digit by digit
// from the top (a histogram of 256 bins each), then each wave lists the kept
// tokens of its own run.
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictParams p) {
  __shared__ int s_hist[256];
  __shared__ int s_wave[kSelectWaves][2];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const int pair = blockIdx.x;
  const int b = pair / p.hkv, h = pair % p.hkv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int len = evict_len(p, b);
  int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.keep;
  if (h == 0 && threadIdx.x == 0) {
    const int n = min(len, p.keep);
    if (p.sl_i64)
      static_cast<int64_t*>(p.new_lens)[b * p.nls] = n;
    else
      static_cast<int32_t*>(p.new_lens)[b * p.nls] = n;
  }
  if (len <= p.keep) {
    for (int j = threadIdx.x; j < p.keep; j += kSelectThreads) kept[j] = j < len ? j : -1;
    return;
  }
  const float* row = p.scores + b * p.scs0 + h * p.scs1;
  const int lo = p.sinks, hi = len - p.recent;  // the tokens to choose from: more than `left` of them
  uint32_t prefix = 0;
  int left = p.keep - p.sinks - p.recent;
  if (left > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSelectThreads) s_hist[i] = 0;
      __syncthreads();
      const uint32_t above = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int t = lo + static_cast<int>(threadIdx.x); t < hi; t += kSelectThreads) {
        const uint32_t key = score_key(row[t]);
        if ((key & above) == prefix) atomicAdd(&s_hist[(key >> shift) & 255u], 1);
      }
      __syncthreads();
      if (wave == 0) {
        // bins from the top, four a lane: the first at which the count reaches `left`
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += s_hist[255 - 4 * lane - i];
        const int incl = wave_inclusive_scan_i32(mine, lane);
        const uint64_t hit = __ballot(incl >= left);
        const int l = __builtin_ctzll(hit);
        if (lane == l) {
          int before = incl - mine;
          int bin = 255 - 4 * lane;
          while (before + s_hist[bin] < left) before += s_hist[bin--];
          s_prefix = prefix | static_cast<uint32_t>(bin) << shift;
          s_left = left - before;
        }
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
    }
  }
  // prefix is the key of the last token taken, of which `left` are taken (left
  // == 0: none is chosen and no key counts)
  const bool some = left > 0;
  const int run = (len + kSelectWaves - 1) / kSelectWaves;
  const int first = wave * run, last = min(first + run, len);
  auto kind = [&](int t) {  // 0: goes, 1: stays, 2: stays while equals are left
    if (t >= last) return 0;
    if (t < lo || t >= hi) return 1;
    const uint32_t key = score_key(row[t]);
    return some ? (key > prefix ? 1 : (key == prefix ? 2 : 0)) : 0;
  };
  int sure = 0, equal = 0;
  for (int t0 = first; t0 < last; t0 += 64) {
    const int k = kind(t0 + lane);
    sure += __popcll(__ballot(k == 1));
    equal += __popcll(__ballot(k == 2));
  }
  if (lane == 0) {
    s_wave[wave][0] = sure;
    s_wave[wave][1] = equal;
  }
  __syncthreads();
  sure = equal = 0;
  for (int x = 0; x < wave; ++x) {
    sure += s_wave[x][0];
    equal += s_wave[x][1];
  }
  const uint64_t below = (uint64_t{1} << lane) - 1;
  for (int t0 = first; t0 < last; t0 += 64) {
    const int k = kind(t0 + lane);
    const uint64_t ms = __ballot(k == 1), me = __ballot(k == 2);
    const int s = sure + __popcll(ms & below), e = equal + __popcll(me & below);
    const int j = s + min(e, left);
    // (j < keep unless the scores change under the launch)
    if ((k == 1 || (k == 2 && e < left)) && j < p.keep) kept[j] = t0 + lane;
    sure += __popcll(ms);
    equal += __popcll(me);
  }
}

// ============================================================== move =====
constexpr int kMoveThreads = 256;

// A source as listed, -1 if it is none of the row's tokens (lengths or scores
// that change under the launches leave rows wrong, and nothing else).
__device__ __forceinline__ int evict_source(const int32_t* kept, int j, int len) {
  const int src = kept[j];
  return static_cast<uint32_t>(src) < static_cast<uint32_t>(len) ? src : -1;
}

// One workgroup per (request, KV head, tensor): K, V or the scores.  V16: rows
// in 16-byte pieces, else element by element (2-byte elements).
template <bool V16>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictParams p) {
  const int pair = blockIdx.x / 3, what = blockIdx.x % 3;
  const int b = pair / p.hkv, h = pair % p.hkv;
  const int len = evict_len(p, b);
  const int n = min(len, p.keep);
  const int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.keep;
  if (what == 2) {
    const float* src = p.scores + b * p.scs0 + h * p.scs1;
    float* dst = p.new_scores + b * p.nss0 + h * p.nss1;
    for (int j0 = 0; j0 < n; j0 += kMoveThreads) {
      const int j = j0 + static_cast<int>(threadIdx.x);
      const int from = j < n ? evict_source(kept, j, len) : -1;
      const float x = from >= 0 ? src[from] : 0.f;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (j < n) dst[j] = x;
    }
    for (int j = n + static_cast<int>(threadIdx.x); j < len; j += kMoveThreads) dst[j] = 0.f;
    return;
  }
  if (len <= p.keep) return;
  using Piece = std::conditional_t<V16, u32x4, uint16_t>;
  char* base = static_cast<char*>(what == 0 ? p.k : p.v);
  const int64_t s0 = what == 0 ? p.ks0 : p.vs0, s1 = what == 0 ? p.ks1 : p.vs1;
  const int64_t s2 = what == 0 ? p.ks2 : p.vs2, s3 = what == 0 ? p.ks3 : p.vs3;
  const int pieces = V16 ? p.head_dim / 8 : p.head_dim;  // of a row: a divisor of the workgroup's threads
  const int64_t step = V16 ? 8 : s3;
  const int piece = threadIdx.x % pieces, rows = kMoveThreads / pieces;
  auto at = [&](int tok) -> char* {
    const int64_t blk = load_index(p.bt, b * p.bts0 + (tok / p.block_size) * p.bts1, p.bt_i64);
    if (blk < 0 || blk >= p.num_blocks) return nullptr;
    return base + 2 * (blk * s0 + h * s1 + (tok % p.block_size) * s2 + piece * step);
  };
  for (int j0 = 0; j0 < n; j0 += rows) {
    const int j = j0 + static_cast<int>(threadIdx.x) / pieces;
    const int src = j < n ? evict_source(kept, j, len) : -1;
    const bool moves = src >= 0 && src != j;
    const char* from = moves ? at(src) : nullptr;
    char* to = moves ? at(j) : nullptr;
    const bool ok = from != nullptr && to != nullptr;
    Piece x{};
    if (ok) x = *reinterpret_cast<const Piece*>(from);
    // the reads have ended, not only begun, before any of the workgroup's writes
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (ok) *reinterpret_cast<Piece*>(to) = x;
  }
}

// ========================================================== host glue ====
namespace {

int evict_params(const fd_kv_evict_args* args, const char* fn, EvictParams& p) {
  if (args == nullptr) return set_error(FD_E_INVALID, "%s: args is NULL", fn);
  const fd_kv_evict_args& a = *args;
  if (a.struct_size != sizeof(fd_kv_evict_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, a.struct_size,
                     sizeof(fd_kv_evict_args));
  if (a.dtype != FD_DTYPE_F16 && a.dtype != FD_DTYPE_BF16)
    return set_error(FD_E_UNSUPPORTED, "%s: dtype must be float16 or bfloat16", fn);
  if (a.num_seqs <= 0 || a.num_kv_heads <= 0 || a.num_blocks <= 0 || a.max_blocks_per_seq <= 0)
    return set_error(FD_E_INVALID, "%s: shapes must be positive", fn);
  if (a.head_dim != 64 && a.head_dim != 128)
    return set_error(FD_E_UNSUPPORTED, "%s: head_dim must be 64 or 128", fn);
  if (a.block_size != 8 && a.block_size != 16 && a.block_size != 32)
    return set_error(FD_E_UNSUPPORTED, "%s: block_size must be 8, 16 or 32", fn);
  if (!a.k_cache || !a.v_cache || !a.block_tables || !a.seq_lens || !a.scores || !a.new_scores || !a.kept ||
      !a.new_seq_lens)
    return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (a.keep < 1 || a.sink_tokens < 0 || a.recent_tokens < 0 || a.sink_tokens + a.recent_tokens > a.keep)
    return set_error(FD_E_INVALID, "%s: keep must be positive and hold sink_tokens and recent_tokens", fn);
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  if (cap > INT32_MAX - kSelectThreads || a.keep > INT32_MAX - kSelectThreads)
    return set_error(FD_E_UNSUPPORTED, "%s: block tables or keep hold 2^31 tokens or more", fn);
  if (a.score_tokens < cap)
    return set_error(FD_E_INVALID, "%s: scores must hold every token of a block-table row", fn);
  if (a.num_seqs * a.num_kv_heads > INT32_MAX / 3) return set_error(FD_E_INVALID, "%s: launch grid too large", fn);
  if (a.new_seq_lens == a.seq_lens)
    return set_error(FD_E_INVALID, "%s: new_seq_lens must not be seq_lens", fn);
  p = EvictParams{};
  p.k = a.k_cache;
  p.ks0 = a.k_stride[0];
  p.ks1 = a.k_stride[1];
  p.ks2 = a.k_stride[2];
  p.ks3 = a.k_stride[3];
  p.v = a.v_cache;
  p.vs0 = a.v_stride[0];
  p.vs1 = a.v_stride[1];
  p.vs2 = a.v_stride[2];
  p.vs3 = a.v_stride[3];
  p.bt = a.block_tables;
  p.bts0 = a.block_tables_stride[0];
  p.bts1 = a.block_tables_stride[1];
  p.bt_i64 = a.block_tables_dtype == FD_INDEX_I64;
  p.sl = a.seq_lens;
  p.sls = a.seq_lens_stride;
  p.sl_i64 = a.seq_lens_dtype == FD_INDEX_I64;
  p.scores = a.scores;
  p.scs0 = a.score_stride[0];
  p.scs1 = a.score_stride[1];
  p.new_scores = a.new_scores;
  p.nss0 = a.new_score_stride[0];
  p.nss1 = a.new_score_stride[1];
  p.kept = a.kept;
  p.new_lens = a.new_seq_lens;
  p.nls = a.new_seq_lens_stride;
  p.hkv = static_cast<int>(a.num_kv_heads);
  p.head_dim = static_cast<int>(a.head_dim);
  p.block_size = static_cast<int>(a.block_size);
  p.cap = static_cast<int>(cap);
  p.keep = static_cast<int>(a.keep);
  p.sinks = static_cast<int>(a.sink_tokens);
  p.recent = static_cast<int>(a.recent_tokens);
  p.num_blocks = a.num_blocks;
  return FD_OK;
}

// Rows in 16-byte pieces: unit dim stride, every row on a 16-byte line.
bool rows_of_16(const fd_kv_evict_args& a) {
  for (const int64_t* s : {a.k_stride, a.v_stride})
    if (s[3] != 1 || s[0] % 8 || s[1] % 8 || s[2] % 8) return false;
  return ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15u) == 0;
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_kv_evict(const fd_kv_evict_args* args, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_kv_evict";
  EvictParams p;
  const int rc = evict_params(args, fn, p);
  if (rc != FD_OK) return rc;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const unsigned pairs = static_cast<unsigned>(args->num_seqs * args->num_kv_heads);
  dispatch(evict_select_kernel, dim3(pairs), dim3(kSelectThreads), stream, nullptr, nullptr, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "evict select launch failed: %s", hipGetErrorString(e));
  rows_of_16(*args) ? dispatch(evict_move_kernel<true>, dim3(3 * pairs), dim3(kMoveThreads), stream, nullptr, nullptr, p)
                    : dispatch(evict_move_kernel<false>, dim3(3 * pairs), dim3(kMoveThreads), stream, nullptr, nullptr, p);
  e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "evict move launch failed: %s", hipGetErrorString(e));
  return FD_OK;
}
