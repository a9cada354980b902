// Single-token decode attention over a 4-bit cache (fp4_format.h), for gfx950.
//
// With s = scale * q.k, x = s log2(e), a row's tokens are cut into chunks of 32-token
// tiles, one a workgroup; each leaves M = max x, L = sum 2^(x - M) and sum 2^(x - M) v,
// and a second launch joins them (join_rows): out = sum_c 2^(M_c - M) acc_c /
// sum_c 2^(M_c - M) L_c.  A row of one chunk is stored at once.
#include "decode_host.h"
#include "fp4_format.h"

namespace fd {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

struct Fp4DecodeParams {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const void* bt;
  const void* sl;
  void* out;
  float* acc;
  float2* stats;
  int64_t qs0, qs1, qs2, ks0, ks1, vs0, vs1, bts0, bts1, sls, os0, os1, os2;
  int bt_i64, sl_i64;
  int hq, hkv, group, block_size, num_blocks, width, chunks, chunk_tiles;
  float scale_log2;
};

// One wave per (request, KV head, up to 8 query heads, chunk); lane = token for q.k,
// lane = dim (pairs of 128-dim heads) for the weighted sum.
constexpr int kFp4Heads = 8;

template <typename T, int D>
__global__ __launch_bounds__(64) void fp4_decode_kernel(Fp4DecodeParams p, int head_blocks) {
  __shared__ float s_q[kFp4Heads][D];
  __shared__ float s_p[kFp4Heads][64];
  __shared__ int64_t s_page[64];  // byte of the token's V block, -1: not attended
  const int lane = threadIdx.x;
  const int chunk = blockIdx.y / head_blocks, hb = blockIdx.y % head_blocks;
  const int b = blockIdx.x / p.hkv, kvh = blockIdx.x % p.hkv;
  const int h0 = hb * kFp4Heads, nh = min(kFp4Heads, p.group - h0);
  const int cap = p.width * p.block_size;
  const int len = min(max(load_index(p.sl, b * p.sls, p.sl_i64), 0), cap);
  const int begin = 32 * chunk * p.chunk_tiles, end = min(begin + 32 * p.chunk_tiles, len);
  if (begin >= end && p.chunks > 1) return;  // the join reads a row's own chunks only

  const T* qb = static_cast<const T*>(p.q) + b * p.qs0;
  for (int i = lane; i < kFp4Heads * D; i += 64) {
    const int j = i / D, d = i % D;
    s_q[j][d] = j < nh ? to_f32(qb[(kvh * p.group + h0 + j) * p.qs1 + d * p.qs2]) : 0.f;
  }
  float m[kFp4Heads], l[kFp4Heads], acc[kFp4Heads][D / 64];
#pragma unroll
  for (int j = 0; j < kFp4Heads; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) acc[j][e] = 0.f;
  }
  __syncthreads();
  for (int t0 = begin; t0 < end; t0 += 64) {
    const int tok = t0 + lane;
    bool ok = tok < end;
    int64_t blk = 0;
    if (ok) {
      blk = load_index(p.bt, b * p.bts0 + (tok / p.block_size) * p.bts1, p.bt_i64);
      ok = blk >= 0 && blk < p.num_blocks;
    }
    const int off = tok % p.block_size;
    float s[kFp4Heads] = {};
    if (ok) {
      const uint8_t* page = p.k + blk * p.ks0 + kvh * p.ks1;
      for (int d = 0; d < D; d += 8) {
        const uint32_t code = *reinterpret_cast<const uint32_t*>(page + fp4_key_at<D>(off, d));
        const float scale =
            __builtin_bit_cast(float, static_cast<uint32_t>(page[fp4_key_scale_at<D>(p.block_size, off, d)]) << 23);
        const f32x2_t x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 2),
                              __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 3)};
#pragma unroll
        for (int j = 0; j < kFp4Heads; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) s[j] += s_q[j][d + e] * x[e / 2][e % 2];
      }
    }
    s_page[lane] = ok ? blk * p.vs0 + kvh * p.vs1 : -1;
#pragma unroll
    for (int j = 0; j < kFp4Heads; ++j) {
      const float x = ok ? s[j] * p.scale_log2 : -INFINITY;
      float mx = x;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, shfl_xor_f32(mx, o));
      const float m_new = fmaxf(m[j], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[j] - m_use), pj = exp2f(x - m_use);
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
      if (s_page[t] < 0) continue;
      const uint8_t* page = p.v + s_page[t];
      const int at = (t0 + t) % p.block_size;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        const int d = lane + 64 * e;
        const uint32_t code = page[fp4_value_at<D>(at, d)];
        const float scale =
            __builtin_bit_cast(float, static_cast<uint32_t>(page[fp4_value_scale_at<D>(p.block_size, at, d)]) << 23);
        const f32x2_t x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0);
        const float v = d % 2 ? x[1] : x[0];
#pragma unroll
        for (int j = 0; j < kFp4Heads; ++j) acc[j][e] += s_p[j][t] * v;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kFp4Heads; ++j) {
    if (j >= nh) break;
    const int qh = kvh * p.group + h0 + j;
    if (p.chunks == 1) {
      const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
      T* dst = static_cast<T*>(p.out) + b * p.os0 + qh * p.os1;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) dst[(lane + 64 * e) * p.os2] = from_f32<T>(acc[j][e] * inv);
    } else {
      const int64_t at = (static_cast<int64_t>(b) * p.hq + qh) * p.chunks + chunk;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) p.acc[at * D + lane + 64 * e] = acc[j][e];
      if (lane == 0) p.stats[at] = float2{m[j], l[j]};
    }
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
  // (the grid's dimensions: KV heads, rows; a row's head blocks times its chunks)
  if (a.num_seqs > 65535 || a.num_q_heads > (1 << 24))
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
}

struct Fp4Plan {
  int64_t head_blocks, chunks, chunk_tiles, acc, stats;  // acc, stats: floats
  int64_t floats() const { return acc + stats; }
};

Fp4Plan plan_for(const fd_fp4_decode_args& a) {
  Fp4Plan s{};
  s.head_blocks = (a.num_q_heads / a.num_kv_heads + kFp4Heads - 1) / kFp4Heads;
  const int64_t tiles = (a.max_blocks_per_seq * a.block_size + 31) / 32;
  const int64_t wgs = a.num_seqs * a.num_kv_heads * s.head_blocks;
  int64_t chunks = (8 * device_cus() + wgs - 1) / wgs;
  chunks = chunks < (tiles + 1) / 2 ? chunks : (tiles + 1) / 2;
  const int64_t most = 65535 / s.head_blocks;
  chunks = chunks < most ? chunks : most;
  chunks = chunks < 1 ? 1 : chunks;
  s.chunk_tiles = (tiles + chunks - 1) / chunks;
  s.chunks = (tiles + s.chunk_tiles - 1) / s.chunk_tiles;
  if (s.chunks > 1) {
    const int64_t rows = a.num_seqs * a.num_q_heads;
    s.acc = rows * s.chunks * a.head_dim;
    s.stats = (2 * rows * s.chunks + 3) & ~int64_t{3};
  }
  return s;
}

int check_plan(const fd_fp4_decode_args& a, const Fp4Plan& s, const char* fn) {
  if (s.head_blocks > 65535 || a.num_seqs * a.num_kv_heads > INT32_MAX / 64 || a.num_seqs * a.num_q_heads > INT32_MAX)
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  return FD_OK;
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
  Fp4DecodeParams p{};
  p.q = a.q;
  p.k = static_cast<const uint8_t*>(a.k_cache);
  p.v = static_cast<const uint8_t*>(a.v_cache);
  p.bt = a.block_tables;
  p.sl = a.seq_lens;
  p.out = a.out;
  p.acc = workspace;
  p.stats = reinterpret_cast<float2*>(workspace + s.acc);
  p.qs0 = a.q_stride[0];
  p.qs1 = a.q_stride[1];
  p.qs2 = a.q_stride[2];
  p.ks0 = a.k_cache_stride[0];
  p.ks1 = a.k_cache_stride[1];
  p.vs0 = a.v_cache_stride[0];
  p.vs1 = a.v_cache_stride[1];
  p.bts0 = a.block_tables_stride[0];
  p.bts1 = a.block_tables_stride[1];
  p.sls = a.seq_lens_stride;
  p.os0 = a.out_stride[0];
  p.os1 = a.out_stride[1];
  p.os2 = a.out_stride[2];
  p.bt_i64 = a.block_tables_dtype == FD_INDEX_I64;
  p.sl_i64 = a.seq_lens_dtype == FD_INDEX_I64;
  p.hq = static_cast<int>(a.num_q_heads);
  p.hkv = static_cast<int>(a.num_kv_heads);
  p.group = p.hq / p.hkv;
  p.block_size = static_cast<int>(a.block_size);
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.width = static_cast<int>(a.max_blocks_per_seq);
  p.chunks = static_cast<int>(s.chunks);
  p.chunk_tiles = static_cast<int>(s.chunk_tiles);
  p.scale_log2 = a.sm_scale * kLog2e;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const dim3 grid(static_cast<unsigned>(a.num_seqs * a.num_kv_heads), static_cast<unsigned>(s.head_blocks * s.chunks));
  const bool bf = a.dtype == FD_DTYPE_BF16;
  auto go = [&](auto kernel) {
    dispatch(kernel, grid, dim3(64), stream, nullptr, nullptr, p, static_cast<int>(s.head_blocks));
  };
  if (a.head_dim == 64)
    bf ? go(fp4_decode_kernel<__bf16, 64>) : go(fp4_decode_kernel<_Float16, 64>);
  else
    bf ? go(fp4_decode_kernel<__bf16, 128>) : go(fp4_decode_kernel<_Float16, 128>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  if (s.chunks == 1) return FD_OK;
  RowJoin j{};
  j.acc = p.acc;
  j.stats = p.stats;
  j.seq_lens = p.sl;
  j.seq_lens_stride = p.sls;
  j.seq_lens_i64 = p.sl_i64;
  j.hkv = p.hkv;
  j.group = p.group;
  j.chunks = p.chunks;
  j.chunk_tiles = p.chunk_tiles;
  j.cap = p.width * p.block_size;
  j.rows = a.num_seqs * a.num_q_heads;
  j.out = a.out;
  for (int i = 0; i < 3; ++i) j.out_stride[i] = a.out_stride[i];
  return join_rows(j, bf, static_cast<int>(a.head_dim), fn, stream);
}
