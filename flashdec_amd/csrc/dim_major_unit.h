// Loads and arithmetic of a 32-token unit of a dim-major cache (device code).
#pragma once

#include "decode_unit.h"

namespace fd {

// ------------------------------------------------- dim-major caches ----
// A dim-major cache ([blocks, KV heads, head_dim, block_size], token stride
// 1) stores a head's block as head_dim rows of block_size tokens.  A 32-token
// unit is read as 16-byte pieces of those rows (eight tokens of one dim), and
// the lane tokens are reordered so that lane 16*g + c scores tokens 8*g + i,
// i < 8 (i = 4*mt + r: row 4*g + r of QK row block mt):
//   K piece i of lane l: dim 16*i + l/4, tokens 8*(l%4) + [0, 8) -- staged
//     through LDS and read back transposed into the QK A operand
//   vf[n] of lane 16*g + c: dim 16*n + c, tokens 8*g + [0, 8) -- already the
//     PV A operand (V^T row 16*n + c, k = the lane's eight tokens); one load
//     instruction reads 16 consecutive dim rows
// (D = 128: K pieces i < 8 and V operands n < 8; D = 64: four of each.)
// A piece lies in one block: quarter q of the unit is in page q (8-token
// blocks), q / 2 (16) or 0 (32).
constexpr int kDmWaves = 4;
constexpr int kDmRowBytes = 64;  // one staged dim row: 32 tokens x 2 bytes

template <int D>
struct DmRegs {
  static constexpr int KS = D / 32;  // QK k-steps
  u32x4 kf[2][KS];                   // raw K pieces, then QK A operands
  u32x4 vf[D / 16];                  // PV A operands
  uint32_t bmask;                    // bit i: token 8*g + i lies in a valid block
};

template <typename T, int BS, bool NT, int D>
__device__ __forceinline__ void load_unit_dm(const DecodeParams& p, int kvh, const UnitPages& up, int lane,
                                             DmRegs<D>& t) {
  constexpr int KS = DmRegs<D>::KS;
  static_assert(BS == 8 || BS == 16 || BS == 32, "dim-major units need 8-, 16- or 32-token blocks");
  constexpr int64_t E = sizeof(T);
  const int q = lane & 3;   // K: the lane's eight-token quarter of the unit
  const int g = lane >> 4;  // V: the lane's eight tokens
  const int c = lane & 15;
  // the block holding quarter x of the unit; invalid ids read block 0
  // (masked at compute time)
  auto page = [&](int x) -> int32_t {
    if constexpr (BS == 32) return up.a;
    else if constexpr (BS == 16) return x < 2 ? up.a : up.b;
    else return x == 0 ? up.a : x == 1 ? up.b : x == 2 ? up.c : up.d;
  };
  auto valid = [&](int32_t blk) { return blk >= 0 && blk < p.num_blocks; };
  const int32_t kpg = page(q);
  const int32_t vpg = page(g);
  const int32_t kblk = valid(kpg) ? kpg : 0;
  const int32_t vblk = valid(vpg) ? vpg : 0;
  const char* kp = static_cast<const char*>(p.k) +
                   (kblk * p.ks0 + kvh * p.ks1 + (lane >> 2) * p.ks3 + (8 * q) % BS) * E;
  const char* vp = static_cast<const char*>(p.v) + (vblk * p.vs0 + kvh * p.vs1 + c * p.vs3 + (8 * g) % BS) * E;
  const int64_t kstep = 16 * p.ks3 * E;
  const int64_t vstep = 16 * p.vs3 * E;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) t.kf[i / KS][i % KS] = kv_load<NT>(kp + i * kstep);
#pragma unroll
  for (int n = 0; n < D / 16; ++n) t.vf[n] = kv_load<NT>(vp + n * vstep);
  t.bmask = valid(vpg) ? 0xffu : 0u;
}

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The unit's raw K pieces go to the wave's LDS stage (row = dim, 64 bytes
// of tokens) and come back as QK A operands: kf[mt][s] of lane 16*g + c =
// token 8*(c/4) + 4*mt + c%4 (A row c), dims 32*s + 8*g + [0, 8).  One
// ds_read_b64_tr_b16 gives lane c of a 16-lane group element j of the
// 8-byte piece addressed by lane 4*j + c/4, element c%4; so lane c' of the
// group addresses dim row base + c'/4 at tokens 8*(c'%4) + 4*mt + [0, 4).
// A wave's LDS operations run in order, so the stage needs no barrier
// between the writes and the reads, nor before the next unit's writes.
//
// Rows 8r .. 8r+7 with r odd hold each 16-byte piece with its two 8-byte
// halves swapped.  The read of a 16-lane group covers the same 8-byte half of
// every piece in four rows; groups g and g + 1 read rows 8 apart, which without
// the swap sit on the same banks (rows 64 bytes apart, 512 bytes per 8 rows).
// Row 16i + lane/4 is odd-eighth exactly for lanes 32..63; read row
// 8g + c/4 (+4, +32s) for odd g.
template <int D>
__device__ __forceinline__ void stage_k_dm(DmRegs<D>& t, uint8_t* stage, int lane) {
  constexpr int KS = DmRegs<D>::KS;
  lds_u8* st = (lds_u8*)stage;
  const bool swap = lane >= 32;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const u32x4 k = t.kf[i / KS][i % KS];
    *(lds_u32x4*)(st + (16 * i + (lane >> 2)) * kDmRowBytes + 16 * (lane & 3)) =
        swap ? u32x4{k[2], k[3], k[0], k[1]} : k;
  }
  const int c = lane & 15;
  const int g = lane >> 4;
  lds_u8* rd = st + (8 * g + (c >> 2)) * kDmRowBytes + 16 * (c & 3);
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      lds_u8* a = rd + 32 * s * kDmRowBytes + 8 * (mt ^ (g & 1));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 4 * kDmRowBytes));
      const u32x2 l2 = __builtin_bit_cast(u32x2, lo);
      const u32x2 h2 = __builtin_bit_cast(u32x2, hi);
      t.kf[mt][s] = u32x4{l2[0], l2[1], h2[0], h2[1]};
    }
  }
}

// Fused append into a dim-major cache: this lane's elements of the new
// token in load_unit_dm's layout -- kd(i) = append_k dim 16*i + lane/4 (its K
// pieces), vd(n) = append_v dim 16*n + c (its V operands), two per register.
template <int D>
struct DmAppendRegs {
  uint32_t k[D / 32];  // element i in bits 16*(i%2) of word i/2
  uint32_t v[D / 32];
  __device__ __forceinline__ uint16_t kd(int i) const { return static_cast<uint16_t>(k[i >> 1] >> (16 * (i & 1))); }
  __device__ __forceinline__ uint16_t vd(int n) const { return static_cast<uint16_t>(v[n >> 1] >> (16 * (n & 1))); }
};

template <typename T, int D>
__device__ __forceinline__ void load_append_dm(const DecodeParams& p, int b, int kvh, int lane,
                                               DmAppendRegs<D>& ar) {
  const uint16_t* ak = static_cast<const uint16_t*>(p.ak) + b * p.aks0 + kvh * p.aks1;
  const uint16_t* av = static_cast<const uint16_t*>(p.av) + b * p.avs0 + kvh * p.avs1;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const int kd = 32 * j + (lane >> 2), vd = 32 * j + (lane & 15);
    ar.k[j] = ak[kd * p.aks2] | (static_cast<uint32_t>(ak[(kd + 16) * p.aks2]) << 16);
    ar.v[j] = av[vd * p.avs2] | (static_cast<uint32_t>(av[(vd + 16) * p.avs2]) << 16);
  }
}

// The new token's K/V go to slot (block, offset) of the dim-major cache: one
// element per dim row.  Lanes with lane % 4 == 0 hold every K dim once, lanes
// with g == 0 every V dim.
template <typename T, int BS, int D>
__device__ __forceinline__ void store_append_dm(const DecodeParams& p, int kvh, int32_t slot, int lane,
                                                const DmAppendRegs<D>& ar) {
  const int64_t blk = slot / BS, off = slot % BS;
  if (blk >= p.num_blocks) return;
  if ((lane & 3) == 0) {
    uint16_t* dst = static_cast<uint16_t*>(p.k) + blk * p.ks0 + kvh * p.ks1 + off * p.ks2;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) dst[(16 * i + (lane >> 2)) * p.ks3] = ar.kd(i);
  }
  if ((lane >> 4) == 0) {
    uint16_t* dst = static_cast<uint16_t*>(p.v) + blk * p.vs0 + kvh * p.vs1 + off * p.vs2;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) dst[(16 * n + lane) * p.vs3] = ar.vd(n);
  }
}

// Element e (a token of the lane's eight) of a 16-byte piece replaced by x.
__device__ __forceinline__ void set_elem16(u32x4& piece, int e, uint16_t x) {
  const int sh = (e & 1) * 16;
  const uint32_t keep = ~(0xffffu << sh);
#pragma unroll
  for (int w = 0; w < 4; ++w)
    piece[w] = (w == (e >> 1)) ? ((piece[w] & keep) | (static_cast<uint32_t>(x) << sh)) : piece[w];
}

// process_unit for a dim-major unit (load_unit_dm's layout): the lane's
// scores and V columns are tokens 8*g + i, and V needs no transposes.
template <typename T, bool FUSE, int D, bool LAZY = true, typename Take = NoScores>
__device__ __forceinline__ void process_unit_dm(DmRegs<D>& t, const u32x4 (&qf)[D / 32], float scale_log2,
                                                int tok0, int first, int last, int app,
                                                const DmAppendRegs<D>& ar, int lane, uint8_t* stage,
                                                WaveState<D>& st, Take take = {}) {
  constexpr int KS = DmRegs<D>::KS;
  constexpr int NTILE = D / 16;
  const int g = lane >> 4;
  uint32_t vmask = t.bmask;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int tok = tok0 + 8 * g + i;
    vmask &= (tok <= last && (first == 0 || tok >= first)) ? ~0u : ~(1u << i);
  }
  if constexpr (FUSE) {
    // the new token comes from registers: token at = 8*qa + e of this unit
    const int at = app - tok0;
    if (at >= 0 && at < 32) {
      const int qa = at >> 3, e = at & 7;
      if ((lane & 3) == qa) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) set_elem16(t.kf[i / KS][i % KS], e, ar.kd(i));
      }
      if (g == qa) {
#pragma unroll
        for (int n = 0; n < NTILE; ++n) set_elem16(t.vf[n], e, ar.vd(n));
        vmask |= 1u << e;
      }
    }
  }
  stage_k_dm<D>(t, stage, lane);
  float sc[8];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    f32x4 sb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) sb = mfma16x16x32<T>(t.kf[mt][s], qf[s], sb);
#pragma unroll
    for (int r = 0; r < 4; ++r) sc[4 * mt + r] = sb[r] * scale_log2;
  }
  // masked tokens: -inf scores and zeroed V elements (word w of every V
  // operand holds tokens 2w and 2w + 1)
  if (__ballot(vmask != 0xffu)) {
    uint32_t keep[4];
#pragma unroll
    for (int w = 0; w < 4; ++w)
      keep[w] = (((vmask >> (2 * w)) & 1u) ? 0x0000ffffu : 0u) | (((vmask >> (2 * w + 1)) & 1u) ? 0xffff0000u : 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] = ((vmask >> i) & 1u) ? sc[i] : -INFINITY;
#pragma unroll
    for (int n = 0; n < NTILE; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w) t.vf[n][w] &= keep[w];
  }
  take(0, sc);
  float pr[8];
  softmax_step<8, D, LAZY>(sc, pr, st);
  u32x4 pp;
#pragma unroll
  for (int j = 0; j < 4; ++j) pp[j] = pack2<T>(pr[2 * j], pr[2 * j + 1]);
#pragma unroll
  for (int n = 0; n < NTILE; ++n) st.acc[n] = mfma16x16x32<T>(t.vf[n], pp, st.acc[n]);
}

}  // namespace fd
