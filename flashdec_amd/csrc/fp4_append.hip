// Appending to a 4-bit cache (fp4_format.h), and reading it back by slot, for gfx950.
//
//   append: q and k of a token are rotated at its position (rope_math.h), q is rounded
//           to its type, k and v are quantised and stored at the token's slot.
//   read:   k and v of a slot as 16-bit values.
//
// Keys are quantised from the 32-bit rotation: a rounding to 16 bits between would
// only add its error.  The rotation's products and sums are rounded one by one, so
// that a table's cos/sin give the same codes everywhere.
#include "decode_host.h"
#include "fp4_format.h"
#include "rope_math.h"

#pragma clang fp contract(off)

namespace fd {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

struct Fp4AppendParams {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  uint8_t* k_cache;
  uint8_t* v_cache;
  const void* block_ids;
  const void* block_offsets;
  const void* positions;
  int64_t qs0, qs1, ks0, ks1, vs0, vs1, os0, os1;  // elements: token, head
  int64_t kcs0, kcs1, vcs0, vcs1;                  // bytes: block, head
  int32_t i64;                                     // bits 0, 1, 2: 64-bit ids, offsets, positions
  int32_t hq, hkv, block_size, rotary_dim;         // hq 0: no rotation
  int32_t per_xcd;                                 // tokens that one XCD takes, neighbours; 0: in turn
  int64_t num_blocks, tokens;
  float base;
  const float* tab;
  int64_t tab_rows;
};

constexpr int kFp4Threads = 256;

// Whether a token's slot lies in the cache; else it is not stored.
__device__ __forceinline__ bool fp4_slot(const Fp4AppendParams& p, int64_t t, int64_t& blk, int& off) {
  // (whole 64-bit values: a wrong index is refused, not cut to one that is in range)
  const int64_t b = p.i64 & 1 ? static_cast<const int64_t*>(p.block_ids)[t] : static_cast<const int32_t*>(p.block_ids)[t];
  const int64_t o =
      p.i64 & 2 ? static_cast<const int64_t*>(p.block_offsets)[t] : static_cast<const int32_t*>(p.block_offsets)[t];
  blk = b;
  off = static_cast<int>(o);
  return b >= 0 && b < p.num_blocks && o >= 0 && o < p.block_size;
}

template <typename T>
__device__ __forceinline__ void fp4_unpack(const u32x4& w, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = lo_f32<T>(w[j]);
    x[2 * j + 1] = hi_f32<T>(w[j]);
  }
}

// Rows that a call reads or writes once do not push out of the caches what others left
// there (8192 tokens appended and read back, over inputs that no cache holds any more:
// 59.8 -> 52.6 us; loads kept and only stores streamed 55.0).  The caller's rows may lie
// off 16-byte lines: the store asks for no more than an element's alignment, and is one
// instruction all the same.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void fp4_stream_out(void* dst, u32x4 x) {
  __builtin_nontemporal_store(x, static_cast<u32x4_any*>(dst));
}

// L = D / 8 lanes a head, eight dims a lane, S heads a workgroup.  Workgroup (x, y)
// takes token x's heads y * S + s: every load that the rows need is under way before
// the first is used, and a token's workgroups are independent.
//   VEC: rows on 16-byte lines and R / 2 a multiple of 8, so that a piece and its
//   partners are a load each (the second mostly hits in L1); else element by element.
//   TABLE: cos/sin from the caller's table, eight of each a lane, for VEC; else through
//   LDS.
// Bound by memory for prompts (8192 tokens, Hq 32, Hkv 8, D 128: 177 MB read and written
// in 42 us, 4.2 TB/s, a large copy's 4.9; K and V alone 14.8), by its dependent loads
// for a step (one token, Hq 16, Hkv 2: 2.8 us).  Element by element 128 us, 2 bytes a load
// or store; without a table 75, as each of a token's workgroups computes its cos and sin.
template <typename T, int D, bool VEC, bool TABLE>
__global__ __launch_bounds__(kFp4Threads) void fp4_append_kernel(Fp4AppendParams p) {
  static_assert(VEC || !TABLE, "tables element by element go through LDS");
  constexpr int L = D / 8;             // lanes a head
  constexpr int S = kFp4Threads / L;   // heads at once
  __shared__ float s_cos[TABLE ? 1 : D / 2], s_sin[TABLE ? 1 : D / 2];
  const int64_t t = xcd_logical_block(blockIdx.x, p.per_xcd);
  if (t >= p.tokens) return;
  const int c = threadIdx.x % L;
  const int half = p.rotary_dim / 2;
  const int r = blockIdx.y * S + threadIdx.x / L;
  const bool there = r < p.hq + 2 * p.hkv;
  const bool is_q = r < p.hq, is_v = r >= p.hq + p.hkv;
  const int h = is_q ? r : (is_v ? r - p.hq - p.hkv : r - p.hq);
  const T* row = is_q   ? static_cast<const T*>(p.q) + t * p.qs0 + h * p.qs1
                 : is_v ? static_cast<const T*>(p.v) + t * p.vs0 + h * p.vs1
                        : static_cast<const T*>(p.k) + t * p.ks0 + h * p.ks1;
  const bool turns = there && !is_v && 8 * c < 2 * half;  // (VEC: all of the piece or none)
  const bool second = 8 * c >= half;
  u32x4 own = {}, other = {};
  if constexpr (VEC) {
    if (there) own = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + 8 * c));
    if (turns) other = *reinterpret_cast<const u32x4*>(row + 8 * c + (second ? -half : half));
  }
  f32x4 cs[4];
  if constexpr (TABLE) {
    const int64_t pos = load_index_uniform(p.positions, t, p.i64 & 4);
    const int64_t at = pos < 0 ? 0 : (pos < p.tab_rows ? pos : p.tab_rows - 1);
    if (turns) {
      const float* tab = p.tab + at * half + 8 * c - (second ? half : 0);
      const float* sin = tab + p.tab_rows * half;
      __builtin_memcpy(&cs[0], tab, 32);
      __builtin_memcpy(&cs[2], sin, 32);
    }
  } else if (p.hq > 0) {
    const int64_t pos = load_index_uniform(p.positions, t, p.i64 & 4);
    for (int i = threadIdx.x; i < half; i += kFp4Threads) {
      if (p.tab != nullptr)
        rope_table_cos_sin(p.tab, p.tab_rows, half, pos, i, s_cos[i], s_sin[i]);
      else
        rope_cos_sin(p.base, p.rotary_dim, pos, i, s_cos[i], s_sin[i]);
    }
    __syncthreads();
  }
  int64_t blk;
  int off;
  const bool stored = fp4_slot(p, t, blk, off);
  if (!there) return;
  float y[8];
  if constexpr (VEC) {
    float x[8], z[8];
    fp4_unpack<T>(own, x);
    fp4_unpack<T>(other, z);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float co = 1.f, si = 0.f;
      if constexpr (TABLE) {
        co = cs[e / 4][e % 4];
        si = cs[2 + e / 4][e % 4];
      } else if (turns) {
        const int i = 8 * c + e - (second ? half : 0);
        co = s_cos[i];
        si = s_sin[i];
      }
      float lo, hi;
      rope_rotate(second ? z[e] : x[e], second ? x[e] : z[e], co, si, lo, hi);
      y[e] = turns ? (second ? hi : lo) : x[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * c + e;
      y[e] = to_f32(row[d]);
      if (!is_v && d < 2 * half) {
        const float z = to_f32(row[d < half ? d + half : d - half]);
        const int i = d < half ? d : d - half;
        float lo, hi;
        rope_rotate(d < half ? y[e] : z, d < half ? z : y[e], s_cos[i], s_sin[i], lo, hi);
        y[e] = d < half ? lo : hi;
      }
    }
  }
  if (is_q) {
    T* dst = static_cast<T*>(p.q_out) + t * p.os0 + h * p.os1 + 8 * c;
    if constexpr (VEC) {
      fp4_stream_out(dst, u32x4{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])});
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = from_f32<T>(y[e]);
    }
    return;
  }
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max(amax, __builtin_bit_cast(uint32_t, y[e]) & 0x7fffffffu);
  // over the four lanes of a group: neighbours, then the pairs
  amax = max(amax, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(amax), 0xb1, 0xf, 0xf, false)));
  amax = max(amax, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(amax), 0x4e, 0xf, 0xf, false)));
  const uint32_t byte = fp4_scale_byte(amax);
  uint32_t code = 0;
  if (byte != kFp4NaN) {
    const float scale = __builtin_bit_cast(float, byte << 23);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[0], y[1], scale, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], scale, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], scale, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], scale, 3);
  }
  if (!stored) return;
  if (!is_v) {
    uint8_t* page = p.k_cache + blk * p.kcs0 + h * p.kcs1;
    *reinterpret_cast<uint32_t*>(page + fp4_key_at<D>(off, 8 * c)) = code;
    if ((c & 3) == 0) page[fp4_key_scale_at<D>(p.block_size, off, 8 * c)] = static_cast<uint8_t>(byte);
  } else {
    uint8_t* page = p.v_cache + blk * p.vcs0 + h * p.vcs1;
    if constexpr (D == 128) {
      *reinterpret_cast<uint32_t*>(page + fp4_value_at<D>(off, 8 * c)) = code;
    } else {
      *reinterpret_cast<uint16_t*>(page + fp4_value_at<D>(off, 8 * c)) = static_cast<uint16_t>(code);
      *reinterpret_cast<uint16_t*>(page + fp4_value_at<D>(off, 8 * c + 4)) = static_cast<uint16_t>(code >> 16);
    }
    if ((c & 3) == 0) page[fp4_value_scale_at<D>(p.block_size, off, 8 * c)] = static_cast<uint8_t>(byte);
  }
}

struct Fp4ReadParams {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  void* k_out;
  void* v_out;
  const void* block_ids;
  const void* block_offsets;
  int64_t kcs0, kcs1, vcs0, vcs1;  // bytes: block, head
  int64_t ks0, ks1, vs0, vs1;      // elements: token, head
  int32_t i64, hkv, block_size;
  int32_t group;                   // tokens of a workgroup
  int64_t num_blocks, tokens;
};

// Eight dims a lane, D / 8 lanes a row; a workgroup takes the 2 hkv rows (K or V, KV
// head) of N groups of tokens, or a part (y) of one's, the loads of all N under way
// together.  Calls that fill the card take N = 4, neighbours, whose values share lines
// (8192 tokens, Hkv 8, D 128, 42 MB: 10.5 us, with N = 1 13.3).
template <typename T, int D, int N>
__global__ __launch_bounds__(kFp4Threads) void fp4_read_kernel(Fp4ReadParams p) {
  constexpr int L = D / 8, S = kFp4Threads / L;
  const int c = threadIdx.x % L, slot = threadIdx.x / L;
  const int heads = 2 * p.hkv;
  const int mine = p.group > 1 ? slot / heads : 0;
  const int rest = p.group > 1 ? slot - mine * heads : static_cast<int>(blockIdx.y) * S + slot;
  if (mine >= p.group || rest >= heads) return;
  const bool is_v = rest >= p.hkv;
  const int h = is_v ? rest - p.hkv : rest;
  const int64_t t0 = blockIdx.x * static_cast<int64_t>(N) * p.group + mine;
  int64_t blk[N], at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t t = min(t0 + i * p.group, p.tokens - 1);
    // (whole 64-bit values: a wrong index is refused, not cut to one that is in range)
    blk[i] = p.i64 & 1 ? static_cast<const int64_t*>(p.block_ids)[t] : static_cast<const int32_t*>(p.block_ids)[t];
    at[i] = p.i64 & 2 ? static_cast<const int64_t*>(p.block_offsets)[t] : static_cast<const int32_t*>(p.block_offsets)[t];
  }
  uint32_t code[N], byte[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool held = blk[i] >= 0 && blk[i] < p.num_blocks && at[i] >= 0 && at[i] < p.block_size;
    const int off = static_cast<int>(at[i]);
    code[i] = 0;
    byte[i] = 2;
    if (!held) continue;
    if (!is_v) {
      const uint8_t* page = p.k_cache + blk[i] * p.kcs0 + h * p.kcs1;
      code[i] = *reinterpret_cast<const uint32_t*>(page + fp4_key_at<D>(off, 8 * c));
      byte[i] = page[fp4_key_scale_at<D>(p.block_size, off, 8 * c)];
    } else {
      const uint8_t* page = p.v_cache + blk[i] * p.vcs0 + h * p.vcs1;
      if constexpr (D == 128) {
        code[i] = *reinterpret_cast<const uint32_t*>(page + fp4_value_at<D>(off, 8 * c));
      } else {
        code[i] = *reinterpret_cast<const uint16_t*>(page + fp4_value_at<D>(off, 8 * c)) |
                  static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(page + fp4_value_at<D>(off, 8 * c + 4))) << 16;
      }
      byte[i] = page[fp4_value_scale_at<D>(p.block_size, off, 8 * c)];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t t = t0 + i * p.group;
    if (t >= p.tokens) return;
    // (the conversion goes by the scale's exponent alone; 255 gives NaN)
    const float scale = __builtin_bit_cast(float, byte[i] << 23);
    const f32x2_t x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[i], scale, 0);
    const f32x2_t x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[i], scale, 1);
    const f32x2_t x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[i], scale, 2);
    const f32x2_t x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[i], scale, 3);
    T* dst = is_v ? static_cast<T*>(p.v_out) + t * p.vs0 + h * p.vs1 : static_cast<T*>(p.k_out) + t * p.ks0 + h * p.ks1;
    fp4_stream_out(dst + 8 * c,
                   u32x4{pack2<T>(x0[0], x0[1]), pack2<T>(x1[0], x1[1]), pack2<T>(x2[0], x2[1]), pack2<T>(x3[0], x3[1])});
  }
}

namespace {

bool aligned(const void* ptr, uintptr_t n) { return (reinterpret_cast<uintptr_t>(ptr) & (n - 1)) == 0; }

}  // namespace

int check_fp4_caches(const char* fn, int64_t head_dim, int64_t block_size, int64_t num_blocks, int64_t num_kv_heads,
                     const void* k_cache, const int64_t* ks, const void* v_cache, const int64_t* vs) {
  if (head_dim != 64 && head_dim != 128)
    return set_error(FD_E_UNSUPPORTED, "%s: head_dim must be 64 or 128", fn);
  if (block_size != 8 && block_size != 16 && block_size != 32)
    return set_error(FD_E_UNSUPPORTED, "%s: block_size must be 8, 16 or 32", fn);
  if (num_blocks <= 0 || num_kv_heads <= 0) return set_error(FD_E_INVALID, "%s: shapes must be positive", fn);
  if (num_blocks > INT32_MAX || num_kv_heads > 65535)
    return set_error(FD_E_UNSUPPORTED, "%s: too many blocks or KV heads", fn);
  if (k_cache == nullptr || v_cache == nullptr) return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return set_error(FD_E_INVALID, "%s: caches must be 16-byte aligned", fn);
  for (const int64_t* st : {ks, vs})
    for (int i = 0; i < 2; ++i)
      if (st[i] < 0 || st[i] % 16 != 0)
        return set_error(FD_E_INVALID, "%s: cache strides must be non-negative multiples of 16 bytes", fn);
  return FD_OK;
}

namespace {

// Whether 16-bit rows of unit dim stride lie on 16-byte lines.
bool on_lines(const void* at, const int64_t* stride) { return aligned(at, 16) && stride[0] % 8 == 0 && stride[1] % 8 == 0; }

template <typename T, int D>
int launch_append(const fd_fp4_append_args& a, Fp4AppendParams p, const char* fn, hipStream_t stream) {
  const int heads = p.hq + 2 * p.hkv, s = kFp4Threads / (D / 8);
  const int64_t parts = (heads + s - 1) / s;
  // Neighbours in the cache share lines, values four tokens a piece, so that many of them
  // go to one XCD and its L2 joins what they write (8192 tokens, Hq 32, Hkv 8, D 128: 92 -> 76 MB
  // written, which is what there is to write, 36.7 -> 35.0 us from warm caches).  Few are
  // spread over all XCDs.
  p.per_xcd = a.num_tokens * parts >= 8 * device_cus() ? static_cast<int32_t>((a.num_tokens + 7) / 8) : 0;
  const dim3 grid(static_cast<unsigned>(p.per_xcd > 0 ? 8 * p.per_xcd : a.num_tokens), static_cast<unsigned>(parts));
  const bool vec = on_lines(a.k, a.k_stride) && on_lines(a.v, a.v_stride) && a.rotary_dim % 16 == 0 &&
                   (p.hq == 0 || (on_lines(a.q, a.q_stride) && on_lines(a.q_out, a.q_out_stride)));
  auto go = [&](auto kernel) {
    if (launch_record_on()) record_launch(reinterpret_cast<const void*>(kernel), stream);
    hipLaunchKernelGGL(kernel, grid, dim3(kFp4Threads), 0, stream, p);
  };
  if (!vec)
    go(fp4_append_kernel<T, D, false, false>);
  else if (p.hq > 0 && p.tab != nullptr)
    go(fp4_append_kernel<T, D, true, true>);
  else
    go(fp4_append_kernel<T, D, true, false>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return FD_OK;
}

template <typename T, int D>
int launch_read(Fp4ReadParams p, const char* fn, hipStream_t stream) {
  const int64_t heads = 2 * p.hkv, rows = kFp4Threads / (D / 8);
  p.group = heads < rows ? static_cast<int32_t>(rows / heads) : 1;
  const int64_t groups = (p.tokens + p.group - 1) / p.group, parts = p.group > 1 ? 1 : (heads + rows - 1) / rows;
  auto go = [&](auto kernel, int64_t n) {
    const dim3 grid(static_cast<unsigned>((groups + n - 1) / n), static_cast<unsigned>(parts));
    if (launch_record_on()) record_launch(reinterpret_cast<const void*>(kernel), stream);
    hipLaunchKernelGGL(kernel, grid, dim3(kFp4Threads), 0, stream, p);
  };
  // (from 16 workgroups a CU on)
  groups * parts >= 16 * device_cus() ? go(fp4_read_kernel<T, D, 4>, 4) : go(fp4_read_kernel<T, D, 1>, 1);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "%s: launch failed: %s", fn, hipGetErrorString(e));
  return FD_OK;
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_fp4_append(const fd_fp4_append_args* args, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_fp4_append";
  if (args == nullptr) return set_error(FD_E_INVALID, "%s: args is NULL", fn);
  const fd_fp4_append_args& a = *args;
  if (a.struct_size != sizeof(fd_fp4_append_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, a.struct_size,
                     sizeof(fd_fp4_append_args));
  if (a.dtype != FD_DTYPE_F16 && a.dtype != FD_DTYPE_BF16)
    return set_error(FD_E_UNSUPPORTED, "%s: dtype must be float16 or bfloat16", fn);
  const int rc = check_fp4_caches(fn, a.head_dim, a.block_size, a.num_blocks, a.num_kv_heads, a.k_cache,
                                  a.k_cache_stride, a.v_cache, a.v_cache_stride);
  if (rc != FD_OK) return rc;
  if (a.num_tokens < 0) return set_error(FD_E_INVALID, "%s: shapes must be positive", fn);
  const bool rope = a.rotary_dim != 0;
  if (a.num_tokens == 0) return FD_OK;
  if (!a.k || !a.v || !a.block_ids || !a.block_offsets) return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  if (rope) {
    if (!a.q || !a.q_out || !a.positions || a.num_q_heads <= 0)
      return set_error(FD_E_INVALID, "%s: a rotation needs q, q_out and positions", fn);
    if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 2 != 0)
      return set_error(FD_E_INVALID, "%s: rotary_dim must be positive, even and <= head_dim", fn);
    if (!(a.base > 0.0) || a.base > 3.4e38)
      return set_error(FD_E_INVALID, "%s: base must be a positive finite number", fn);
    if (a.cos_sin_table != nullptr && (a.table_rows <= 0 || !aligned(a.cos_sin_table, 4)))
      return set_error(FD_E_INVALID, "%s: cos_sin_table needs table_rows > 0 and 4-byte alignment", fn);
    if (a.num_q_heads > 65535) return set_error(FD_E_UNSUPPORTED, "%s: too many query heads", fn);
  }
  // (2^32 - 1 threads along the grid's first dimension)
  if (a.num_tokens > INT64_C(0xffffffff) / kFp4Threads - 8)
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  Fp4AppendParams p{};
  p.tokens = a.num_tokens;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_out = a.q_out;
  p.k_cache = static_cast<uint8_t*>(a.k_cache);
  p.v_cache = static_cast<uint8_t*>(a.v_cache);
  p.block_ids = a.block_ids;
  p.block_offsets = a.block_offsets;
  p.positions = a.positions;
  p.qs0 = a.q_stride[0];
  p.qs1 = a.q_stride[1];
  p.ks0 = a.k_stride[0];
  p.ks1 = a.k_stride[1];
  p.vs0 = a.v_stride[0];
  p.vs1 = a.v_stride[1];
  p.os0 = a.q_out_stride[0];
  p.os1 = a.q_out_stride[1];
  p.kcs0 = a.k_cache_stride[0];
  p.kcs1 = a.k_cache_stride[1];
  p.vcs0 = a.v_cache_stride[0];
  p.vcs1 = a.v_cache_stride[1];
  for (int i = 0; i < 3; ++i) p.i64 |= a.index_dtype[i] == FD_INDEX_I64 ? 1 << i : 0;
  p.hq = rope ? static_cast<int32_t>(a.num_q_heads) : 0;
  p.hkv = static_cast<int32_t>(a.num_kv_heads);
  p.block_size = static_cast<int32_t>(a.block_size);
  p.rotary_dim = static_cast<int32_t>(a.rotary_dim);
  p.num_blocks = a.num_blocks;
  p.base = static_cast<float>(a.base);
  p.tab = a.cos_sin_table;
  p.tab_rows = a.table_rows;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const bool bf = a.dtype == FD_DTYPE_BF16;
  if (a.head_dim == 64) return bf ? launch_append<__bf16, 64>(a, p, fn, stream) : launch_append<_Float16, 64>(a, p, fn, stream);
  return bf ? launch_append<__bf16, 128>(a, p, fn, stream) : launch_append<_Float16, 128>(a, p, fn, stream);
}

extern "C" int fd_fp4_read(const fd_fp4_read_args* args, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_fp4_read";
  if (args == nullptr) return set_error(FD_E_INVALID, "%s: args is NULL", fn);
  const fd_fp4_read_args& a = *args;
  if (a.struct_size != sizeof(fd_fp4_read_args))
    return set_error(FD_E_INVALID, "%s: struct_size %u != %zu (ABI mismatch)", fn, a.struct_size,
                     sizeof(fd_fp4_read_args));
  if (a.dtype != FD_DTYPE_F16 && a.dtype != FD_DTYPE_BF16)
    return set_error(FD_E_UNSUPPORTED, "%s: dtype must be float16 or bfloat16", fn);
  const int rc = check_fp4_caches(fn, a.head_dim, a.block_size, a.num_blocks, a.num_kv_heads, a.k_cache,
                                  a.k_cache_stride, a.v_cache, a.v_cache_stride);
  if (rc != FD_OK) return rc;
  if (a.num_tokens < 0) return set_error(FD_E_INVALID, "%s: shapes must be positive", fn);
  if (a.num_tokens == 0) return FD_OK;
  if (!a.k_out || !a.v_out || !a.block_ids || !a.block_offsets)
    return set_error(FD_E_INVALID, "%s: NULL tensor pointer", fn);
  // (2^32 - 1 threads along the grid's first dimension)
  if (a.num_tokens > INT64_C(0xffffffff) / kFp4Threads)
    return set_error(FD_E_UNSUPPORTED, "%s: launch grid too large", fn);
  Fp4ReadParams p{};
  p.k_cache = static_cast<const uint8_t*>(a.k_cache);
  p.v_cache = static_cast<const uint8_t*>(a.v_cache);
  p.k_out = a.k_out;
  p.v_out = a.v_out;
  p.block_ids = a.block_ids;
  p.block_offsets = a.block_offsets;
  p.kcs0 = a.k_cache_stride[0];
  p.kcs1 = a.k_cache_stride[1];
  p.vcs0 = a.v_cache_stride[0];
  p.vcs1 = a.v_cache_stride[1];
  p.ks0 = a.k_out_stride[0];
  p.ks1 = a.k_out_stride[1];
  p.vs0 = a.v_out_stride[0];
  p.vs1 = a.v_out_stride[1];
  for (int i = 0; i < 2; ++i) p.i64 |= a.index_dtype[i] == FD_INDEX_I64 ? 1 << i : 0;
  p.hkv = static_cast<int32_t>(a.num_kv_heads);
  p.block_size = static_cast<int32_t>(a.block_size);
  p.num_blocks = a.num_blocks;
  p.tokens = a.num_tokens;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const bool bf = a.dtype == FD_DTYPE_BF16;
  if (a.head_dim == 64) return bf ? launch_read<__bf16, 64>(p, fn, stream) : launch_read<_Float16, 64>(p, fn, stream);
  return bf ? launch_read<__bf16, 128>(p, fn, stream) : launch_read<_Float16, 128>(p, fn, stream);
}
