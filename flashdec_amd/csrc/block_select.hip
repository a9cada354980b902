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
#include "decode_host.h"

namespace fd {

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

// Both of a and b, NaN where either is.
__device__ __forceinline__ float min_nan(float a, float b) { return a < b || a != a ? a : b; }
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }

// Workgroup (i, head, row): the row's i-th block with new tokens that is complete; a
// thread a dim.
template <typename T>
__global__ __launch_bounds__(128) void key_bounds_kernel(BoundsParams p) {
  const int b = blockIdx.z, h = blockIdx.y, d = threadIdx.x;
  const int64_t cap = static_cast<int64_t>(p.width) * p.block_size;
  int64_t len = load_index(p.sl, b * p.sls, p.sl_i64);
  len = len < 0 ? 0 : (len < cap ? len : cap);
  const int64_t first = (len > p.new_tokens ? len - p.new_tokens : 0) / p.block_size;
  const int64_t at = first + blockIdx.x;
  if (at >= len / p.block_size || d >= p.head_dim) return;
  const int64_t blk = load_index(p.bt, b * p.bts0 + at * p.bts1, p.bt_i64);
  if (blk < 0 || blk >= p.num_blocks) return;
  const T* k = static_cast<const T*>(p.k) + blk * p.ks0 + h * p.ks1 + d * p.ks3;
  float lo = to_f32(k[0]), hi = lo;
  for (int t = 1; t < p.block_size; ++t) {
    const float x = to_f32(k[t * p.ks2]);
    lo = min_nan(lo, x);
    hi = max_nan(hi, x);
  }
  T* dst = static_cast<T*>(p.bounds) + (blk * p.hkv + h) * 2 * p.head_dim + d;
  dst[0] = from_f32<T>(lo);
  dst[p.head_dim] = from_f32<T>(hi);
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
  int bt_i64, sl_i64, hkv, group, block_size, width, select, sinks, recent;
  int64_t num_blocks, block_step;  // block_step: a pool block's distance in KV-head blocks
};

// A row's length and blocks.
struct SelectRow {
  int64_t len;
  int blocks;
};
__device__ __forceinline__ SelectRow select_row(const SelectParams& p, int b) {
  const int64_t cap = static_cast<int64_t>(p.width) * p.block_size;
  int64_t len = load_index(p.sl, b * p.sls, p.sl_i64);
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

// A wave a block: lanes share the dims.
template <typename T, int D>
__global__ __launch_bounds__(256) void block_score_kernel(SelectParams p) {
  const int pair = blockIdx.y, b = pair / p.hkv, h = pair % p.hkv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const SelectRow r = select_row(p, b);
  if (r.blocks <= p.select) return;  // all of them
  double up[D / 64], down[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) up[e] = down[e] = 0.0;
  for (int g = 0; g < p.group; ++g) {
    const T* q = static_cast<const T*>(p.q) + b * p.qs0 + (h * p.group + g) * p.qs1;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      const double x = to_f32(q[(lane + 64 * e) * p.qs2]);
      up[e] += x < 0 ? 0.0 : x;  // (a NaN goes into both)
      down[e] += x > 0 ? 0.0 : x;
    }
  }
  const int last = r.blocks - p.recent;
  for (int j = p.sinks + blockIdx.x * 4 + wave; j < last; j += gridDim.x * 4) {
    const int64_t blk = load_index(p.bt, b * p.bts0 + j * p.bts1, p.bt_i64);
    uint32_t key = 0;
    if (blk >= 0 && blk < p.num_blocks) {
      const T* lo = static_cast<const T*>(p.bounds) + (blk * p.hkv + h) * 2 * D;
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        s += up[e] * to_f32(lo[D + lane + 64 * e]);
        s += down[e] * to_f32(lo[lane + 64 * e]);
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      key = score_key(s);
    }
    if (lane == 0) p.keys[static_cast<int64_t>(pair) * p.width + j] = key;
  }
}

constexpr int kPickThreads = 256;

// Exclusive sum over the workgroup, and the whole sum.
__device__ __forceinline__ int pick_scan(int x, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = wave_inclusive_scan_i32(x, lane);
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; ++w) {
    before += w < wave ? s_wave[w] : 0;
    total += s_wave[w];
  }
  __syncthreads();
  return before + upto - x;
}

// A workgroup a (request, KV head): the key that the chosen ones reach, eight bits at a
// time, then the chosen blocks in their order.
__global__ __launch_bounds__(kPickThreads) void block_pick_kernel(SelectParams p) {
  __shared__ int s_count[256], s_wave[kPickThreads / 64], s_digit, s_left;
  const int pair = blockIdx.x, b = pair / p.hkv, h = pair % p.hkv, tid = threadIdx.x;
  const SelectRow r = select_row(p, b);
  const bool all = r.blocks <= p.select;
  const uint32_t* keys = p.keys + static_cast<int64_t>(pair) * p.width;
  const int first = p.sinks, last = r.blocks - p.recent;
  uint32_t least = 0;  // the least key chosen
  int left = p.select - p.sinks - p.recent;
  if (!all) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_count[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int j = first + tid; j < last; j += kPickThreads)
        if ((keys[j] & mask) == least) atomicAdd(&s_count[(keys[j] >> shift) & 255], 1);
      __syncthreads();
      // thread t: digit 255 - t, and how many keys have a larger one
      const int mine = s_count[255 - tid];
      int total;
      const int above = pick_scan(mine, s_wave, total);
      if (above < left && above + mine >= left) {
        s_digit = 255 - tid;
        s_left = left - above;
      }
      __syncthreads();
      least |= left > 0 ? static_cast<uint32_t>(s_digit) << shift : 255u << shift;
      left = left > 0 ? s_left : 0;
    }
  }
  // `left` of the keys that equal `least` are chosen, the lowest blocks first
  int32_t* blocks = p.blocks + static_cast<int64_t>(pair) * p.select;
  int32_t* tables = p.tables + static_cast<int64_t>(pair) * p.select;
  int n = 0, equal = 0;
  for (int j0 = 0; j0 < r.blocks; j0 += kPickThreads) {
    const int j = j0 + tid;
    const bool there = j < r.blocks, always = there && (all || j < first || j >= last);
    const uint32_t key = there && !always ? keys[j] : 0u;
    const bool ties = there && !always && key == least;
    int total;
    const int rank = equal + pick_scan(ties ? 1 : 0, s_wave, total);
    equal += total;
    const bool chosen = always || (there && !always && key > least) || (ties && rank < left);
    const int at = n + pick_scan(chosen ? 1 : 0, s_wave, total);
    n += total;
    if (chosen) {
      const int64_t blk = load_index(p.bt, b * p.bts0 + j * p.bts1, p.bt_i64);
      blocks[at] = j;
      tables[at] = blk >= 0 && blk < p.num_blocks ? static_cast<int32_t>(blk * p.block_step + h) : -1;
    }
  }
  for (int i = n + tid; i < p.select; i += kPickThreads) blocks[i] = tables[i] = -1;
  // (the row's last block, which may be partly filled, is always chosen)
  if (tid == 0)
    p.lens[pair] = static_cast<int32_t>(static_cast<int64_t>(n) * p.block_size -
                                        (static_cast<int64_t>(r.blocks) * p.block_size - r.len));
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

int64_t select_words(const fd_block_select_args& a) { return a.num_seqs * a.num_kv_heads * a.max_blocks_per_seq; }

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
  if (!a.k_cache || !a.block_tables || !a.seq_lens || !a.bounds) return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (reinterpret_cast<uintptr_t>(a.bounds) & 15u) return set_error(FD_E_INVALID, "%s: bounds must be 16-byte aligned", fn);
  // blocks that the new tokens of a row may complete
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  const int64_t fresh = a.new_tokens < cap ? a.new_tokens : cap;
  const int64_t touched = (fresh + a.block_size - 1) / a.block_size;
  if (touched == 0) return FD_OK;
  if (!grid_fits(touched, 128)) return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
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
  const dim3 grid(static_cast<unsigned>(touched), static_cast<unsigned>(a.num_kv_heads), static_cast<unsigned>(a.num_seqs));
  const dim3 block(static_cast<unsigned>(a.head_dim));
  if (a.dtype == FD_DTYPE_BF16)
    dispatch(key_bounds_kernel<__bf16>, grid, block, stream, nullptr, nullptr, p);
  else
    dispatch(key_bounds_kernel<_Float16>, grid, block, stream, nullptr, nullptr, p);
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
  if (workspace == nullptr || words < select_words(a) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
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
  p.bt_i64 = a.block_tables_dtype == FD_INDEX_I64;
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
  if (a.max_blocks_per_seq > a.select) {  // else every row has all of its blocks
    int64_t parts = (8 * device_cus() + pairs - 1) / pairs;
    const int64_t most = (a.max_blocks_per_seq + 3) / 4;
    parts = parts < most ? parts : most;
    const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(pairs));
    auto score = [&](auto kernel) { dispatch(kernel, grid, dim3(256), stream, nullptr, nullptr, p); };
    const bool bf = a.dtype == FD_DTYPE_BF16;
    if (a.head_dim == 64)
      bf ? score(block_score_kernel<__bf16, 64>) : score(block_score_kernel<_Float16, 64>);
    else
      bf ? score(block_score_kernel<__bf16, 128>) : score(block_score_kernel<_Float16, 128>);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  }
  dispatch(block_pick_kernel, dim3(static_cast<unsigned>(pairs)), dim3(kPickThreads), stream, nullptr, nullptr, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return FD_OK;
}
