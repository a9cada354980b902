// Eviction from a paged K/V cache by accumulated attention weight, for gfx950.
//
// A row of len > keep tokens keeps its first `sinks`, its last `recent` and, of
// the tokens between, the keep - sinks - recent of highest score, in their order:
//   kept = sort(sinks u recent u top(score)),  K'[j] = K[kept[j]], V', score' alike.
// Ties go to the lower index; NaN ranks below every number and -0 equals 0.
//
// kept[j] >= j, so entries are moved in place: the places [j0, j1) are sources of
// entries in front of j1 only, of at most j1 - j0 consecutive ones.  A workgroup
// that has read its own chunk of entries may write it once the (at most two) lower
// chunks that read from these places have read theirs.
#include "decode_host.h"

namespace fd {

constexpr int kTurnLine = 32;  // words of a cache line

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
  // words of the workspace: per pair the length; the next chunk to be taken, on a cache
  // line of its own, and for every chunk whether it has been read; per 64 tokens how
  // many of those in front are kept
  int32_t* lens;
  uint32_t* turns;
  int32_t* ranks;
  int chunks, turn_words, rank_words;
  int bt_i64, sl_i64;
  int hkv, head_dim, block_size, cap;
  int keep, sinks, recent;
  int64_t num_blocks;
};

__device__ __forceinline__ int evict_len(const EvictParams& p, int b) {
  const int n = load_index(p.sl, b * p.sls, p.sl_i64);
  return n < 0 ? 0 : (n < p.cap ? n : p.cap);
}

// Order of the scores as unsigned integers: NaN 1, then -inf .. +inf, the two
// zeros alike.  Two more keys stand for tokens that are not chosen from: none for
// no token, all for one that stays in any case.
constexpr uint32_t kKeyNone = 0u, kKeyAll = ~0u;

__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 + 0 = 0
  const uint32_t key = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  return x != x ? 1u : key;
}

// ============================================================ select =====
constexpr int kSelectThreads = 1024;
constexpr int kSelectMost = 32;  // keys a thread
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kBinBits = 12;  // of a pass: four bins a thread
constexpr int kBins = 1 << kBinBits, kMyBins = kBins / kSelectThreads;
static_assert(kMyBins == 4 && kSelectWaves == 16);
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Inclusive sum over the wave's lanes: shifts within each 16-lane row, then the row
// totals carried across.
__device__ __forceinline__ int select_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// Of one number a wave, x[wave * step]: the sum in front of this wave's (first) and of all.
struct SelectSums {
  int first, all;
};
__device__ __forceinline__ SelectSums select_sums(const int* x, int step, int wave, int lane) {
  const int own = x[step * (lane & 15)];  // (every row of 16 lanes alike)
  int sum = own;
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xf, 0xf, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xf, 0xf, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xf, 0xf, true);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xf, 0xf, true);
  return SelectSums{__builtin_amdgcn_readlane(sum - own, wave), __builtin_amdgcn_readlane(sum, 15)};
}

// Largest of the wave's lanes, in lane 63.
template <int CTRL, int ROWS, bool ZERO>
__device__ __forceinline__ uint32_t select_max_step(uint32_t x) {
  const int y = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, ZERO);
  return max(x, static_cast<uint32_t>(y));
}
__device__ __forceinline__ uint32_t select_max(uint32_t x) {
  x = select_max_step<0x111, 0xf, true>(x);
  x = select_max_step<0x112, 0xf, true>(x);
  x = select_max_step<0x114, 0xf, true>(x);
  x = select_max_step<0x118, 0xf, true>(x);
  x = select_max_step<0x142, 0xa, false>(x);
  return select_max_step<0x143, 0xc, false>(x);
}

// One workgroup per (request, KV head).  The key of the last token chosen is found
// by narrowing a range of keys: from the least to the largest there is, cut into
// 4096 equal bins, to the bin that holds it, until all of a bin is taken or it
// holds one key: two passes for scores that spread over a few octaves, three at
// most.  Then the kept tokens are listed in order.  E: keys a thread holds in
// registers, 64 E consecutive tokens of a batch of 1024 E in each wave, so that a
// wave counts its own runs of 64 and 16 counts are summed.  ONE: rows of one batch;
// others read their scores again in every pass.
// Bound by latency, and for long rows by the one CU's issue rate.  16 rows of 2048
// tokens 5.3 us, of which the scores' trip 0.6, extremes 0.5, a pass 1.0 and 0.8,
// the list 0.8; 16 rows of 32768 17.1: 1.5, 1.7, 3.9 and 1.8, 4.2.  (Digits of 8
// bits from the top, where most scores share the first two: 34 us for the latter.)
template <int E, bool ONE>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictParams p) {
  constexpr int kBatch = kSelectThreads * E;
  __shared__ __attribute__((aligned(16))) int s_bin[kBins];
  __shared__ int s_wave[kSelectWaves];
  __shared__ uint32_t s_least[kSelectWaves], s_most[kSelectWaves];
  __shared__ int s_found[3];  // bin, tokens in it, tokens to take from it
  __shared__ int s_kept[kSelectWaves][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pair = blockIdx.x;
  const int b = pair / p.hkv, h = pair - b * p.hkv;
  const int len = evict_len(p, b);
  int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.keep;
  if (tid == 0) {
    p.lens[pair] = len;
    p.turns[static_cast<int64_t>(pair) * p.turn_words] = 0u;
    if (h == 0) {
      const int n = min(len, p.keep);
      if (p.sl_i64)
        static_cast<int64_t*>(p.new_lens)[b * p.nls] = n;
      else
        static_cast<int32_t*>(p.new_lens)[b * p.nls] = n;
    }
  }
  if (len <= p.keep) {
    for (int j = tid; j < p.keep; j += kSelectThreads) kept[j] = j < len ? j : -1;
    return;
  }
  const float* row = p.scores + b * p.scs0 + h * p.scs1;
  const int lo = p.sinks, hi = len - p.recent;  // the tokens to choose from: more than `left` of them
  const int batches = ONE ? 1 : (len + kBatch - 1) / kBatch;
  uint32_t key[E];
  const int wave0 = 64 * E * wave;  // the wave's first token in a batch
  auto load = [&](int t0) {
    const int at = t0 + wave0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t t = min(at + 64 * e + lane, len - 1);
      key[e] = __builtin_bit_cast(uint32_t, row[t]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = score_key(__builtin_bit_cast(float, key[e]));
    if (at >= lo && at + 64 * E <= hi) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int t = at + 64 * e + lane;
      key[e] = t < lo || t >= hi ? (t < len ? kKeyAll : kKeyNone) : key[e];
    }
  };
  load(0);
  for (int c = tid; c < p.chunks; c += kSelectThreads) p.turns[static_cast<int64_t>(pair) * p.turn_words + kTurnLine + c] = 0u;
#pragma unroll
  for (int i = 0; i < kMyBins; ++i) s_bin[kSelectThreads * i + tid] = 0;
  int left = p.keep - p.sinks - p.recent;
  // chosen: every key from `sure` up, and `left` of the tokens whose key is `last`
  // (kKeyAll - 1: no token's)
  uint32_t sure = kKeyAll, last = kKeyAll - 1;
  if (left > 0) {
    // the largest of -key and of key + 1: kKeyNone and kKeyAll wrap round and drop out
    uint32_t least = 0u, most = 0u;
    for (int x = 0; x < batches; ++x) {
      if (batches > 1) load(kBatch * x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        least = max(least, 0u - key[e]);
        most = max(most, key[e] + 1);
      }
    }
    least = select_max(least);
    most = select_max(most);
    if (lane == 63) {
      s_least[wave] = least;
      s_most[wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) {
      least = max(least, s_least[w]);
      most = max(most, s_most[w]);
    }
    least = 0u - least;
    --most;
    for (;;) {
      const uint32_t range = most - least;
      const int bits = range == 0 ? 0 : 32 - __builtin_clz(range);
      const int shift = bits > kBinBits ? bits - kBinBits : 0;  // range >> shift < kBins
      for (int x = 0; x < batches; ++x) {
        if (batches > 1) load(kBatch * x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t at = key[e] - least;
          if (at <= range) atomicAdd(&s_bin[at >> shift], 1);
        }
      }
      __syncthreads();
      // thread t has the t-th four bins from the top
      i32x4& bins = *reinterpret_cast<i32x4*>(&s_bin[kBins - kMyBins * (tid + 1)]);
      const i32x4 held_by = bins;
      bins = i32x4{0, 0, 0, 0};
      const int mine = held_by[0] + held_by[1] + held_by[2] + held_by[3];
      int incl = select_scan(mine);
      if (lane == 63) s_wave[wave] = incl;
      if (tid < 3) s_found[tid] = 0;
      __syncthreads();
      incl += select_sums(s_wave, 1, wave, lane).first;
      int before = incl - mine;
      if (incl >= left && before < left) {
#pragma unroll
        for (int i = kMyBins - 1; i >= 0; --i) {
          if (before < left && before + held_by[i] >= left) {
            s_found[0] = kBins - kMyBins * (tid + 1) + i;
            s_found[1] = held_by[i];
            s_found[2] = left - before;
          }
          before += held_by[i];
        }
      }
      __syncthreads();
      const uint32_t bin = s_found[0];
      const int held = s_found[1];
      left = s_found[2];
      least += bin << shift;
      if (held == left) {  // all of the bin (or none, if the scores change under the launch)
        sure = least;
        left = 0;
        break;
      }
      if (shift == 0) {
        last = least;
        sure = last + 1;
        break;
      }
      const uint32_t top = least + ((1u << shift) - 1);
      most = top < most ? top : most;
    }
  }
  // The tokens in order: those that stay for sure, and of the equals the first `left`.
  sure = __builtin_amdgcn_readfirstlane(sure);
  last = __builtin_amdgcn_readfirstlane(last);
  left = __builtin_amdgcn_readfirstlane(left);
  int sure_before = 0, equal_before = 0;  // in front of the batch
  for (int x = 0; x < batches; ++x) {
    if (batches > 1) load(kBatch * x);
    int stays = 0, equals = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      stays += __popcll(__ballot(key[e] >= sure));
      equals += __popcll(__ballot(key[e] == last));
      // (counted here: all ballots ahead of their counts do not fit the scalar registers)
      asm volatile("" : "+s"(stays), "+s"(equals));
    }
    if (x > 0) __syncthreads();
    if (lane == 0) {
      s_kept[wave][0] = stays;
      s_kept[wave][1] = equals;
    }
    __syncthreads();
    const SelectSums sures = select_sums(&s_kept[0][0], 2, wave, lane), same = select_sums(&s_kept[0][1], 2, wave, lane);
    int s0 = sure_before + sures.first, e0 = equal_before + same.first;  // in front of the run of 64 tokens
    sure_before += sures.all;
    equal_before += same.all;
    // (opaque, so that the ballots above are not kept for below, nor the lanes' numbers
    // compared ahead of the loop: 4 E and 2 E registers)
    int at = lane;
    asm volatile("" : "+s"(sure), "+s"(last), "+v"(at));
    const int t0 = kBatch * x + wave0;
    int rank = 0;  // lane e: kept tokens in front of run e
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t stay = __ballot(key[e] >= sure), equal = __ballot(key[e] == last);
      const int before = s0 + min(e0, left);
      rank = at == e ? before : rank;
      bool take = key[e] >= sure;
      int j;
      if (equal == 0 || e0 >= left) {
        j = before;
      } else {
        const int e1 = e0 + __builtin_amdgcn_mbcnt_hi(equal >> 32, __builtin_amdgcn_mbcnt_lo(equal, 0));
        j = s0 + min(e1, left);
        take = take || (key[e] == last && e1 < left);
      }
      j = __builtin_amdgcn_mbcnt_hi(stay >> 32, __builtin_amdgcn_mbcnt_lo(stay, j));
      // (j < keep unless the scores change under the launch)
      if (take && j < p.keep) kept[static_cast<uint32_t>(j)] = t0 + 64 * e + lane;
      s0 += __popcll(stay);
      e0 += __popcll(equal);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (lane < E && t0 + 64 * lane < len) p.ranks[static_cast<int64_t>(pair) * p.rank_words + (t0 >> 6) + lane] = rank;
  }
}

// ============================================================== move =====
// Entries of a workgroup of so many threads: 128 bytes of K and V a thread.  A row's
// workgroups take their turns from one counter and those of few rows are few, so
// large jobs have large workgroups.  Us for 256 / 512 threads: 2 pairs of 512
// entries of 128 dims 6.6 / 7.2, 16 of 1024 9.1 / 9.5, 256 of 2560 107 / 105, 16 of
// 8192 of 64 dims 20.5 / 18.0 (and 24.0 with half the entries a thread).
constexpr int kMoveThreads = 256;
__host__ __device__ constexpr int evict_chunk(int head_dim, int threads) { return threads * 32 / head_dim; }

// A source as listed, -1 if it is none of the row's tokens (lengths or scores
// that change under the launches leave rows wrong, and nothing else).
__device__ __forceinline__ int evict_source(const int32_t* kept, int j, int len) {
  const int src = kept[j];
  return static_cast<uint32_t>(src) < static_cast<uint32_t>(len) ? src : -1;
}

// Says that the workgroup's reads for `chunk` have ended, and waits for the lower
// chunks among those of the entries [k0, k1), which read where it will write.
template <int CHUNK>
__device__ __forceinline__ void evict_turn(uint32_t* turn, int chunk, int k0, int k1) {
  uint32_t* done = turn + kTurnLine;
  const int tid = threadIdx.x;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) __hip_atomic_store(&done[chunk], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (tid < 64) {
    // (ranks of another launch's making: still a lower chunk, or none)
    const int first = max(k0, 0) / CHUNK, last = min((k1 - 1) / CHUNK, chunk - 1);
    for (int c = first + tid; c <= last; c += 64)
      while (__hip_atomic_load(&done[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0u) __builtin_amdgcn_s_sleep(2);
  }
  __syncthreads();
}

// Rows in 16-byte pieces: one workgroup per chunk of entries, both tensors and the
// scores.  Its reads go out at once and are waited for, then it says that they are
// done, waits for the lower chunks that read where it writes, and writes.  The
// chunks of a row are taken in turn (a counter), so that whoever waits, waits for
// workgroups that have started and that wait for nothing before they say so: every
// wait ends, in whatever order the workgroups come.  No data passes between
// workgroups, so the flags need no fences: a read whose data has arrived is over.
// Bound by HBM reads and writes (256 pairs of 2560 entries of 128 dims: 105 us, 4.9
// TB/s of both, a large copy's rate), in small jobs by five dependent trips: length
// and turn, list, block ids, rows, the lower chunks' flags.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void evict_move_kernel(EvictParams p) {
  constexpr int kChunk = evict_chunk(D, THREADS);
  constexpr int kPieces = D / 8, kRows = THREADS / kPieces, kIter = kChunk / kRows;
  __shared__ int s_chunk;
  const int tid = threadIdx.x;
  const int pair = blockIdx.x / p.chunks;
  const int b = pair / p.hkv, h = pair - b * p.hkv;
  uint32_t* turn = p.turns + static_cast<int64_t>(pair) * p.turn_words;
  // (the chunk and the length are asked for together; a row that stays needs no chunk)
  if (tid == 0) s_chunk = __hip_atomic_fetch_add(turn, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int len = p.lens[pair];
  const float* score = p.scores + b * p.scs0 + h * p.scs1;
  float* new_score = p.new_scores + b * p.nss0 + h * p.nss1;
  if (len <= p.keep) {
    const int t = (blockIdx.x - pair * p.chunks) * kChunk + tid;
    if (score != new_score && tid < kChunk && t < len) new_score[t] = score[t];
    return;
  }
  __syncthreads();
  const int chunk = s_chunk, n = p.keep, j0 = chunk * kChunk;  // chunk < p.chunks: as many as the row's workgroups
  const int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.keep;
  const int32_t* ranks = p.ranks + static_cast<int64_t>(pair) * p.rank_words;
  // the entries that read from [j0, j0 + kChunk): [k0, k1)
  const int j1 = j0 + kChunk;
  const int k0 = ranks[j0 >> 6], k1 = j1 < len ? ranks[j1 >> 6] : n;

  const int piece = tid % kPieces;
  const int64_t row = static_cast<int64_t>(b) * p.bts0;
  const int shift = 31 - __builtin_clz(p.block_size);  // 8, 16 or 32
  int src[kIter], from_page[kIter], to_page[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int j = j0 + kRows * i + tid / kPieces;
    src[i] = j < n ? evict_source(kept, j, len) : -1;
  }
  const int js = j0 + tid;
  const int score_src = tid < kChunk && js < n ? evict_source(kept, js, len) : -1;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int j = j0 + kRows * i + tid / kPieces;
    const bool moves = src[i] >= 0 && src[i] != j;
    to_page[i] = moves ? load_index(p.bt, row + static_cast<int64_t>(j >> shift) * p.bts1, p.bt_i64) : -1;
    from_page[i] = moves ? load_index(p.bt, row + static_cast<int64_t>(src[i] >> shift) * p.bts1, p.bt_i64) : -1;
  }
  const float score_value = score_src >= 0 ? score[score_src] : 0.f;
  // where the row's tokens behind its new length become this workgroup's to clear:
  // from its first source to the next workgroup's
  const int clear0 = max(n, chunk == 0 ? 0 : evict_source(kept, min(j0, n - 1), len));
  const int clear1 = j1 < n ? evict_source(kept, j1, len) : len;
  u32x4 x[kIter][2];
  bool ok[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    ok[i] = from_page[i] >= 0 && from_page[i] < p.num_blocks && to_page[i] >= 0 && to_page[i] < p.num_blocks;
    const int64_t blk = ok[i] ? from_page[i] : 0, off = ok[i] ? src[i] & (p.block_size - 1) : 0;
    const char* k = static_cast<const char*>(p.k) + 2 * (blk * p.ks0 + h * p.ks1 + off * p.ks2) + 16 * piece;
    const char* v = static_cast<const char*>(p.v) + 2 * (blk * p.vs0 + h * p.vs1 + off * p.vs2) + 16 * piece;
    if (ok[i]) {
      x[i][0] = kv_load<true>(k);
      x[i][1] = kv_load<true>(v);
    }
  }
  evict_turn<kChunk>(turn, chunk, k0, k1);
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    if (!ok[i]) continue;
    const int j = j0 + kRows * i + tid / kPieces;
    const int64_t blk = to_page[i], off = j & (p.block_size - 1);
    *reinterpret_cast<u32x4*>(static_cast<char*>(p.k) + 2 * (blk * p.ks0 + h * p.ks1 + off * p.ks2) + 16 * piece) = x[i][0];
    *reinterpret_cast<u32x4*>(static_cast<char*>(p.v) + 2 * (blk * p.vs0 + h * p.vs1 + off * p.vs2) + 16 * piece) = x[i][1];
  }
  if (tid < kChunk && js < n) new_score[js] = score_value;
  for (int t = clear0 + tid; t < clear1; t += THREADS) new_score[t] = 0.f;
}

// The same for dim-major caches, where a block holds rows of its tokens, one a dim: a
// piece is eight entries of one dim, which lie together where they go (one store) and
// are gathered from where they come from (eight loads of an element, which a wave's
// neighbours mostly find in the same lines).
// Bound by HBM: a line holds the same dim of 32 or 64 tokens, so a row is read nearly
// whole however few of its tokens stay.  32 rows of 4096 tokens to 1024, Hkv 8, D 128:
// 0.54 GB read and 0.13 written in 146 us, 4.6 TB/s (an element at a time by one
// workgroup a row, head and tensor: about 715 us).
template <int D>
__global__ __launch_bounds__(kMoveThreads, 4) void evict_move_dm_kernel(EvictParams p) {
  constexpr int kChunk = evict_chunk(D, kMoveThreads), kGroups = kChunk / 8;
  constexpr int kPieces = D * kGroups / kMoveThreads;  // a thread's, of a tensor
  __shared__ int s_chunk;
  __shared__ int64_t s_from[2][kChunk], s_to[2][kGroups];  // elements from the cache's start
  __shared__ uint32_t s_moves[kGroups];                    // which of a group's entries move
  const int tid = threadIdx.x;
  const int pair = blockIdx.x / p.chunks;
  const int b = pair / p.hkv, h = pair - b * p.hkv;
  uint32_t* turn = p.turns + static_cast<int64_t>(pair) * p.turn_words;
  if (tid == 0) s_chunk = __hip_atomic_fetch_add(turn, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int len = p.lens[pair];
  const float* score = p.scores + b * p.scs0 + h * p.scs1;
  float* new_score = p.new_scores + b * p.nss0 + h * p.nss1;
  if (len <= p.keep) {
    const int t = (blockIdx.x - pair * p.chunks) * kChunk + tid;
    if (score != new_score && tid < kChunk && t < len) new_score[t] = score[t];
    return;
  }
  __syncthreads();
  const int chunk = s_chunk, n = p.keep, j0 = chunk * kChunk, j1 = j0 + kChunk;
  const int32_t* kept = p.kept + static_cast<int64_t>(pair) * p.keep;
  const int32_t* ranks = p.ranks + static_cast<int64_t>(pair) * p.rank_words;
  const int k0 = ranks[j0 >> 6], k1 = j1 < len ? ranks[j1 >> 6] : n;
  const int64_t row = static_cast<int64_t>(b) * p.bts0;
  const int shift = 31 - __builtin_clz(p.block_size), mask = p.block_size - 1;
  float score_value = 0.f;
  const int js = j0 + tid;
  if (tid < kChunk) {
    const int src = js < n ? evict_source(kept, js, len) : -1;
    const bool moves = src >= 0 && src != js;
    const int to = js < n ? load_index(p.bt, row + static_cast<int64_t>(js >> shift) * p.bts1, p.bt_i64) : -1;
    const int from = moves ? load_index(p.bt, row + static_cast<int64_t>(src >> shift) * p.bts1, p.bt_i64) : -1;
    if (src >= 0) score_value = score[src];
    const bool there = to >= 0 && to < p.num_blocks, ok = there && from >= 0 && from < p.num_blocks;
    const int64_t blk = ok ? from : 0, off = ok ? src & mask : 0, dst = there ? to : 0;
    s_from[0][tid] = blk * p.ks0 + h * p.ks1 + off;
    s_from[1][tid] = blk * p.vs0 + h * p.vs1 + off;
    const uint64_t which = __ballot(ok);
    if ((tid & 7) == 0) {
      s_to[0][tid >> 3] = dst * p.ks0 + h * p.ks1 + (js & mask);
      s_to[1][tid >> 3] = dst * p.vs0 + h * p.vs1 + (js & mask);
      s_moves[tid >> 3] = (which >> (tid & 56)) & 0xffu;
    }
  }
  const int clear0 = max(n, chunk == 0 ? 0 : evict_source(kept, min(j0, n - 1), len));
  const int clear1 = j1 < n ? evict_source(kept, j1, len) : len;
  __syncthreads();
  const int group = tid % kGroups, dim0 = tid / kGroups;
  constexpr int kDims = kMoveThreads / kGroups;  // between a thread's pieces
  const uint32_t moves = s_moves[group];
  u32x4 x[2][kPieces];
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const uint16_t* cache = static_cast<const uint16_t*>(what == 0 ? p.k : p.v);
    const int64_t step = what == 0 ? p.ks3 : p.vs3;
    if (moves == 0) continue;
    const uint16_t* from[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) from[e] = cache + s_from[what][8 * group + e] + dim0 * step;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[what][i][e] = from[2 * e][i * kDims * step] | static_cast<uint32_t>(from[2 * e + 1][i * kDims * step]) << 16;
  }
  evict_turn<kChunk>(turn, chunk, k0, k1);
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const int64_t step = what == 0 ? p.ks3 : p.vs3;
    uint16_t* to = static_cast<uint16_t*>(what == 0 ? p.k : p.v) + s_to[what][group] + dim0 * step;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      uint16_t* at = to + i * kDims * step;
      if (moves == 0xffu) {
        *reinterpret_cast<u32x4*>(at) = x[what][i];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (moves >> e & 1u) at[e] = static_cast<uint16_t>(x[what][i][e >> 1] >> (16 * (e & 1)));
      }
    }
  }
  if (tid < kChunk && js < n) new_score[js] = score_value;
  for (int t = clear0 + tid; t < clear1; t += kMoveThreads) new_score[t] = 0.f;
}

// Rows of any strides and alignment, element by element (2-byte elements): one
// workgroup per (request, KV head, tensor), K, V or the scores, front to back.
__global__ __launch_bounds__(kMoveThreads) void evict_move_generic_kernel(EvictParams p) {
  const int pair = blockIdx.x / 3, what = blockIdx.x % 3;
  const int b = pair / p.hkv, h = pair % p.hkv;
  const int len = p.lens[pair];
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
  uint16_t* base = static_cast<uint16_t*>(what == 0 ? p.k : p.v);
  const int64_t s0 = what == 0 ? p.ks0 : p.vs0, s1 = what == 0 ? p.ks1 : p.vs1;
  const int64_t s2 = what == 0 ? p.ks2 : p.vs2, s3 = what == 0 ? p.ks3 : p.vs3;
  const int dim = threadIdx.x % p.head_dim, rows = kMoveThreads / p.head_dim;
  auto at = [&](int tok) -> uint16_t* {
    const int64_t blk = load_index(p.bt, b * p.bts0 + (tok / p.block_size) * p.bts1, p.bt_i64);
    if (blk < 0 || blk >= p.num_blocks) return nullptr;
    return base + blk * s0 + h * s1 + (tok % p.block_size) * s2 + dim * s3;
  };
  for (int j0 = 0; j0 < n; j0 += rows) {
    const int j = j0 + static_cast<int>(threadIdx.x) / p.head_dim;
    const int src = j < n ? evict_source(kept, j, len) : -1;
    const bool moves = src >= 0 && src != j;
    const uint16_t* from = moves ? at(src) : nullptr;
    uint16_t* to = moves ? at(j) : nullptr;
    const bool ok = from != nullptr && to != nullptr;
    const uint16_t x = ok ? *from : uint16_t{0};
    // the reads have ended, not only begun, before any of the workgroup's writes
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (ok) *to = x;
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
  if (a.keep < 1 || a.sink_tokens < 0 || a.recent_tokens < 0 || a.sink_tokens > a.keep ||
      a.recent_tokens > a.keep - a.sink_tokens)
    return set_error(FD_E_INVALID, "%s: keep must be positive and hold sink_tokens and recent_tokens", fn);
  // (blocks of a row first: their tokens may not wrap)
  const int64_t cap = a.max_blocks_per_seq > INT32_MAX ? INT64_MAX : a.max_blocks_per_seq * a.block_size;
  if (cap > INT32_MAX - kSelectThreads * kSelectMost || a.keep > INT32_MAX - kSelectThreads)
    return set_error(FD_E_UNSUPPORTED, "%s: block tables or keep hold 2^31 tokens, or nearly", fn);
  if (a.score_tokens < cap)
    return set_error(FD_E_INVALID, "%s: scores must hold every token of a block-table row", fn);
  if (a.num_seqs > INT32_MAX || a.num_kv_heads > INT32_MAX || a.num_seqs * a.num_kv_heads > INT32_MAX / 3)
    return set_error(FD_E_INVALID, "%s: launch grid too large", fn);
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
  const int64_t most = a.keep < cap ? a.keep : cap;  // entries of a row
  const int chunk = evict_chunk(p.head_dim, kMoveThreads);
  p.chunks = static_cast<int>((most + chunk - 1) / chunk);
  p.turn_words = kTurnLine + (p.chunks + kTurnLine - 1) / kTurnLine * kTurnLine;
  p.rank_words = static_cast<int>((cap + 63) / 64);
  return FD_OK;
}

int64_t evict_up(int64_t words) { return (words + kTurnLine - 1) / kTurnLine * kTurnLine; }
int64_t evict_words(const fd_kv_evict_args& a, const EvictParams& p) {
  const int64_t pairs = a.num_seqs * a.num_kv_heads;
  return evict_up(pairs) + pairs * (static_cast<int64_t>(p.turn_words) + p.rank_words);
}

// Rows in 16-byte pieces: unit dim stride, every row on a 16-byte line.
bool rows_of_16(const fd_kv_evict_args& a) {
  for (const int64_t* s : {a.k_stride, a.v_stride})
    if (s[3] != 1 || s[0] % 8 || s[1] % 8 || s[2] % 8) return false;
  return ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15u) == 0;
}

// Dim-major blocks whose dims' rows lie on 16-byte lines.
bool dims_of_16(const fd_kv_evict_args& a) {
  for (const int64_t* s : {a.k_stride, a.v_stride})
    if (s[2] != 1 || s[0] % 8 || s[1] % 8 || s[3] % 8) return false;
  return ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & 15u) == 0;
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_kv_evict_words(const fd_kv_evict_args* args, int64_t* words) {
  static const char* fn = "fd_kv_evict_words";
  EvictParams p;
  const int rc = evict_params(args, fn, p);
  if (rc != FD_OK) return rc;
  if (words == nullptr) return set_error(FD_E_INVALID, "%s: words is NULL", fn);
  *words = evict_words(*args, p);
  return FD_OK;
}

extern "C" int fd_kv_evict(const fd_kv_evict_args* args, int32_t* workspace, int64_t words, fd_stream_t stream_) {
  clear_launch_record();
  static const char* fn = "fd_kv_evict";
  EvictParams p;
  const int rc = evict_params(args, fn, p);
  if (rc != FD_OK) return rc;
  const int64_t pairs = args->num_seqs * args->num_kv_heads;
  const int64_t need = evict_words(*args, p);
  if (workspace == nullptr || words < need || (reinterpret_cast<uintptr_t>(workspace) & 3u))
    return set_error(FD_E_INVALID, "%s: needs a workspace of %lld words", fn, static_cast<long long>(need));
  p.lens = workspace;
  p.turns = reinterpret_cast<uint32_t*>(workspace + evict_up(pairs));
  p.ranks = workspace + evict_up(pairs) + pairs * p.turn_words;
  // (the workspace has room for the smaller workgroups' chunks)
  const bool rows = rows_of_16(*args), dims = !rows && dims_of_16(*args), large = rows && pairs * p.chunks > device_cus();
  if (large) p.chunks = (p.chunks + 1) / 2;
  const int move_threads = large ? 2 * kMoveThreads : kMoveThreads;
  const int64_t move_grid = pairs * (rows || dims ? p.chunks : 3);
  // (both, before the first launch writes lengths and lists)
  if (!grid_fits(pairs, kSelectThreads) || !grid_fits(move_grid, move_threads))
    return set_error(FD_E_INVALID, "%s: launch grid too large", fn);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  auto select = [&](auto kernel) {
    dispatch(kernel, dim3(static_cast<unsigned>(pairs)), dim3(kSelectThreads), stream, nullptr, nullptr, p);
  };
  // registers for the longest row that the tables hold, as far as they go
  if (p.cap <= 4 * kSelectThreads)
    select(evict_select_kernel<4, true>);
  else if (p.cap <= 16 * kSelectThreads)
    select(evict_select_kernel<16, true>);
  else if (p.cap <= kSelectMost * kSelectThreads)
    select(evict_select_kernel<kSelectMost, true>);
  else
    select(evict_select_kernel<kSelectMost, false>);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "evict select launch failed: %s", hipGetErrorString(e));
  auto move = [&](auto kernel) {
    dispatch(kernel, dim3(static_cast<unsigned>(move_grid)), dim3(static_cast<unsigned>(move_threads)), stream, nullptr,
             nullptr, p);
  };
  if (dims)
    p.head_dim == 128 ? move(evict_move_dm_kernel<128>) : move(evict_move_dm_kernel<64>);
  else if (!rows)
    move(evict_move_generic_kernel);
  else if (large)
    p.head_dim == 128 ? move(evict_move_kernel<128, 2 * kMoveThreads>) : move(evict_move_kernel<64, 2 * kMoveThreads>);
  else
    p.head_dim == 128 ? move(evict_move_kernel<128, kMoveThreads>) : move(evict_move_kernel<64, kMoveThreads>);
  e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_E_LAUNCH, "evict move launch failed: %s", hipGetErrorString(e));
  return FD_OK;
}
