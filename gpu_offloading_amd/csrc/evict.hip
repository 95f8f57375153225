// Eviction of single tokens from a paged cache, per sequence and KV head: the
// `recent` last tokens and those of the largest scores stay, `keep` in all.
//
// Keys are cached with their rotary phase, so attention does not care which slot
// a token sits in: a token that stays in a slot at or above `keep` moves into the
// slot of one that goes below it (ascending to ascending), and nothing else moves.
// At most min(keep, n - keep) rows per head are read and written; sources and
// destinations are disjoint, so the moves need no order.
//
// evict_select_kernel: a workgroup per (sequence, KV head) ranks its tokens by
// (recent, score, lower slot first) with a radix select over 32-bit keys and
// writes the move list.  evict_move_kernel: K, V, score and position of each move,
// bound by memory (rows of one head, 256 bytes at head_dim 128, from anywhere).
#include "kvc_common.h"

#include <algorithm>

namespace kvc {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kPage = 16;
constexpr int kBins = 2048;              // 11 bits of the key at a time, then 11 and 10
// Tokens whose keys are kept in LDS beside the histogram, by the kernel's size;
// longer sequences read them from memory in every pass.
constexpr int kShortKeys = 2048, kMiddleKeys = 8192, kLongKeys = 32768;
constexpr uint32_t kRecentKey = 0xffffffffu, kNanKey = 0xfffffffeu;

struct EvictArgs {
  uint8_t* k_cache;
  uint8_t* v_cache;
  int64_t num_blocks, block_bytes, token_bytes;   // byte strides
  int32_t row_bytes;                              // one head of one token
  int32_t num_kv_heads;
  float* scores;                                  // [num_blocks][Hkv][16]
  int32_t* positions;                             // the same, may be null
  const int32_t* table;
  int64_t table_stride;
  int32_t table_width, table_rows;
  const int32_t* seq_ids;                         // row of the table, may be null
  const int32_t* seq_lens;
  const int32_t* keep;
  const int32_t* recent;
  const int32_t* offsets;                         // may be null
  int32_t batch, max_len, max_moves;
  int32_t* counts;                                // [batch][Hkv] moves
  int32_t* dst;                                   // [batch][Hkv][max_moves] token rows of the
  int32_t* src;                                   // cache (block * 16 + slot), -1: missing
};

__device__ __forceinline__ const int32_t* table_row(const EvictArgs& a, int b) {
  const int row = a.seq_ids ? a.seq_ids[b] : b;
  return row >= 0 && row < a.table_rows ? a.table + row * a.table_stride : nullptr;
}

// The cache's token row of a slot, or -1 where its page is missing.
__device__ __forceinline__ int32_t token_row(const EvictArgs& a, const int32_t* row, int slot) {
  const int32_t id = row[slot / kPage];
  return id >= 0 && id < a.num_blocks ? id * kPage + slot % kPage : -1;
}
__device__ __forceinline__ int64_t score_at(const EvictArgs& a, int32_t token, int h) {
  return (int64_t(token / kPage) * a.num_kv_heads + h) * kPage + token % kPage;
}

// Scores as unsigned keys of the same order; -0 is 0, every NaN ranks above inf.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) return kNanKey;
  const uint32_t u = __float_as_uint(s + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of v over the workgroup's threads before this one.
template <int kThreads>
__device__ __forceinline__ int block_scan(int v, int* wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) wave_sums[wave] = x;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) before += w < wave ? wave_sums[w] : 0;
  return before + x - v;
}

// kKeys: tokens whose keys fit in LDS (0: none are kept).  Bound by latency: the loads, the
// histogram (its atomics meet in few bins where scores are alike; with 11 bits
// rather than 8 in the first pass a bin is a quarter of a power of two) and three
// scans of the keys in which each wave counts its own run of slots by ballots.
template <int kThreads, int kKeys>
__global__ __launch_bounds__(kThreads) void evict_select_kernel(EvictArgs a) {
  constexpr int kWaves = kThreads / 64;
  constexpr bool kLds = kKeys > 0;
  __shared__ alignas(16) uint32_t lds_keys[kLds ? kKeys : 4];
  __shared__ int hist[kBins];
  __shared__ int sums[3][kWaves];
  __shared__ int found[3];
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* row = table_row(a, b);
  const int n = row ? min(min(a.seq_lens[b], a.max_len), a.table_width * kPage) : 0;
  const int keep = min(max(a.keep[b], 0), n);
  int* count = a.counts + int64_t(b) * a.num_kv_heads + h;
  if (n <= keep || keep == 0) {
    if (threadIdx.x == 0) *count = 0;
    return;
  }
  const int offset = a.positions && a.offsets ? a.offsets[b] : 0;
  const int32_t recent_from = int32_t(min(max(int64_t(n) + offset - max(a.recent[b], 0),
                                              int64_t(INT32_MIN)), int64_t(INT32_MAX)));
  // Keys of four slots of one page from s on (the states' rows of 16 are 64-byte
  // aligned), given the token row of the first.  Slots at or past n get 0.
  auto keys_of = [&](int s, int32_t token, f32x4_t f, i32x4_t p) __attribute__((always_inline)) {
    u32x4_t k;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int32_t place = a.positions ? p[e] : s + e;
      k[e] = token < 0 || s + e >= n ? 0u   // a missing page's tokens rank last
             : place >= recent_from  ? kRecentKey : score_key(f[e]);
    }
    return k;
  };
  auto scores_at = [&](int32_t token) __attribute__((always_inline)) {   // (block 0 if missing)
    return *reinterpret_cast<const f32x4_t*>(a.scores + score_at(a, max(token, 0), h));
  };
  auto places_at = [&](int32_t token) __attribute__((always_inline)) {
    return a.positions ? *reinterpret_cast<const i32x4_t*>(a.positions +
                                                           score_at(a, max(token, 0), h))
                       : i32x4_t{0, 0, 0, 0};
  };
  // The pages' first token rows, which the histogram's LDS holds after the selection.
  constexpr int kPages = kLds ? (kKeys / kPage + kThreads - 1) / kThreads : 1;
  static_assert(kKeys / kPage <= kBins, "the pages fit where the histogram was");
  int32_t page[kPages];
  if (kLds) {
#pragma unroll
    for (int i = 0; i < kPages; ++i) {
      const int s = (i * kThreads + int(threadIdx.x)) * kPage;
      page[i] = s < n ? token_row(a, row, s) : -1;
    }
    constexpr int kBatch = 4;   // page ids, then scores, in flight per thread
    for (int s0 = 4 * threadIdx.x; s0 < n; s0 += 4 * kThreads * kBatch) {
      int32_t token[kBatch];
      f32x4_t f[kBatch];
      i32x4_t p[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + 4 * kThreads * i;
        token[i] = s < n ? token_row(a, row, s) : -1;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        f[i] = scores_at(token[i]);
        p[i] = places_at(token[i]);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + 4 * kThreads * i;
        if (s < n) *reinterpret_cast<u32x4_t*>(lds_keys + s) = keys_of(s, token[i], f[i], p[i]);
      }
    }
  }
  auto key4 = [&](int s) __attribute__((always_inline)) {   // s a multiple of 4, below n
    if (kLds) return *reinterpret_cast<const u32x4_t*>(lds_keys + s);
    const int32_t token = token_row(a, row, s);
    return keys_of(s, token, scores_at(token), places_at(token));
  };
  auto key = [&](int s) __attribute__((always_inline)) -> uint32_t {
    if (kLds) return lds_keys[s];
    const int32_t token = token_row(a, row, s);
    if (token < 0) return 0u;
    const int64_t at = score_at(a, token, h);
    return (a.positions ? a.positions[at] : s) >= recent_from ? kRecentKey
                                                              : score_key(a.scores[at]);
  };

  // Radix select of the keep-th largest key: `prefix` holds its bits found so far,
  // `want` how many keys with that prefix stay.
  uint32_t prefix = 0;
  int want = keep;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
    const int shift = kShift[pass];
    for (int i = threadIdx.x; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << kBits[pass]) - 1;
    for (int s = 4 * threadIdx.x; s < n; s += 4 * kThreads) {
      const u32x4_t k = key4(s);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // With the prefix taken off, the keys that have it are at most the mask.
        const uint32_t d = pass == 0 ? k[e] >> shift : (k[e] - prefix) >> shift;
        if (d <= mask && s + e < n) atomicAdd(&hist[d], 1);
      }
    }
    __syncthreads();
    // Bins from the top, kBins / kThreads consecutive ones a thread.
    constexpr int kPer = kBins / kThreads;
    int c[kPer], mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      c[i] = hist[kBins - 1 - (kPer * int(threadIdx.x) + i)];
      mine += c[i];
    }
    int above = block_scan<kThreads>(mine, sums[0]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (above < want && want <= above + c[i]) {
        found[0] = kBins - 1 - (kPer * int(threadIdx.x) + i);
        found[1] = want - above;
        found[2] = c[i];
      }
      above += c[i];
    }
    __syncthreads();
    prefix |= uint32_t(found[0]) << shift;
    want = found[1];
  }

  // Keys above `prefix` stay, and the first `want` equal to it by slot: all of them,
  // mostly.  Wave w has the slots [w run, (w + 1) run).
  const bool rank_ties = found[2] != want;
  const int run = (n + 4 * kThreads - 1) / (4 * kThreads) * 256;
  const int first = min(n, wave * run), last = min(n, first + run);
  auto below = [&](uint64_t m) __attribute__((always_inline)) {
    return int(__builtin_amdgcn_mbcnt_hi(uint32_t(m >> 32),
                                         __builtin_amdgcn_mbcnt_lo(uint32_t(m), 0)));
  };
  auto before = [&](const int* x) __attribute__((always_inline)) {
    int t = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += w < wave ? x[w] : 0;
    return t;
  };
  int ties_before = 0;
  if (rank_ties) {
    int ties = 0;
    for (int s0 = first; s0 < last; s0 += 64) {
      const int s = s0 + lane;
      ties += __builtin_popcountll(
          __builtin_amdgcn_ballot_w64(s < last && key(s) == prefix));
    }
    if (lane == 0) sums[0][wave] = ties;
    __syncthreads();
    ties_before = before(sums[0]);
  }
  // The run's holes and sources, 64 slots at a time and kStep of these in flight:
  // calls put(list, index, slot, mask) where there are any.
  int32_t* dst = a.dst + (int64_t(b) * a.num_kv_heads + h) * a.max_moves;
  int32_t* src = a.src + (int64_t(b) * a.num_kv_heads + h) * a.max_moves;
  auto walk = [&](int holes, int sources, auto put) __attribute__((always_inline)) {
    constexpr int kStep = 4;
    int ties = ties_before;
    for (int s1 = first; s1 < last; s1 += 64 * kStep) {
      uint32_t k[kStep];
#pragma unroll
      for (int g = 0; g < kStep; ++g) k[g] = key(min(s1 + 64 * g + lane, last - 1));
#pragma unroll
      for (int g = 0; g < kStep; ++g) {
        const int s0 = s1 + 64 * g, s = s0 + lane;
        if (s0 >= last) break;
        bool stays = k[g] >= prefix;
        if (rank_ties) {
          const uint64_t tie = __builtin_amdgcn_ballot_w64(s < last && k[g] == prefix);
          stays = k[g] > prefix || (k[g] == prefix && ties + below(tie) < want);
          ties += __builtin_popcountll(tie);
        }
        if (s0 < keep) {
          const uint64_t m = __builtin_amdgcn_ballot_w64(!stays && s < min(keep, last));
          put(dst, holes, s, m);
          holes += __builtin_popcountll(m);
        }
        if (s0 + 63 >= keep) {
          const uint64_t m = __builtin_amdgcn_ballot_w64(stays && s >= keep && s < last);
          put(src, sources, s, m);
          sources += __builtin_popcountll(m);
        }
      }
    }
    return make_int2(holes, sources);
  };
  if (kLds) {
#pragma unroll
    for (int i = 0; i < kPages; ++i)
      if (i * kThreads + threadIdx.x < kBins) hist[i * kThreads + threadIdx.x] = page[i];
  }
  int2 mine = make_int2(0, 0);
  if (rank_ties) {
    mine = walk(0, 0, [](int32_t*, int, int, uint64_t) {});
  } else {
    // Four slots a lane, counted in the lane.
    int low = 0, high = 0;    // tokens that stay below and above `keep`
    for (int s0 = first; s0 < last; s0 += 256) {
      const int s = s0 + 4 * lane;
      if (s >= last) continue;
      const u32x4_t k = key4(s);
      if (s0 + 256 <= min(keep, last)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) low += k[e] >= prefix;
      } else if (s0 >= keep && s0 + 256 <= last) {
#pragma unroll
        for (int e = 0; e < 4; ++e) high += k[e] >= prefix;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          low += s + e < min(keep, last) && k[e] >= prefix;
          high += s + e >= keep && s + e < last && k[e] >= prefix;
        }
      }
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) {
      low += __shfl_xor(low, x);
      high += __shfl_xor(high, x);
    }
    mine = make_int2(max(0, min(keep, last) - first) - low, high);
  }
  if (lane == 0) {
    sums[1][wave] = mine.x;
    sums[2][wave] = mine.y;
  }
  __syncthreads();
  const int hole0 = before(sums[1]);
  walk(hole0, before(sums[2]),
       [&](int32_t* list, int at, int s, uint64_t m) __attribute__((always_inline)) {
         if (!(m >> lane & 1)) return;
         if (kLds) {
           const int32_t token = hist[s / kPage];
           list[at + below(m)] = token < 0 ? -1 : token + s % kPage;
         } else {
           list[at + below(m)] = token_row(a, row, s);
         }
       });
  if (wave == kWaves - 1 && lane == 0) *count = hole0 + mine.x;
}

constexpr int kMoveThreads = 256;
constexpr int64_t kMoveWorkgroups = 4096;   // about; each loops over its share

// 2 * row_bytes / 16 threads per move (K's pieces, then V's), kAhead moves of a
// thread in flight.  64 sequences of 512 to 4096 tokens cut to 1024, 8 heads of 128
// bf16: 268 MB in 56 us, 4.8 TB/s (a large device copy reaches 5.1, copies of whole
// blocks 6.4).
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int kAhead = 4;
  const int h = blockIdx.y % a.num_kv_heads, b = blockIdx.y / a.num_kv_heads;
  const int64_t list = int64_t(b) * a.num_kv_heads + h;
  const int count = a.counts[list];
  const int32_t* dst = a.dst + list * a.max_moves;
  const int32_t* src = a.src + list * a.max_moves;
  const int chunks = a.row_bytes / 16;
  const int lanes = 2 * chunks;
  auto row_at = [&](int32_t token, int piece) __attribute__((always_inline)) {
    return int64_t(token / kPage) * a.block_bytes + int64_t(token % kPage) * a.token_bytes +
           int64_t(h) * a.row_bytes + (piece < chunks ? piece : piece - chunks) * 16;
  };
  const int64_t all = int64_t(count) * lanes, step = int64_t(gridDim.x) * kMoveThreads;
  for (int64_t id0 = int64_t(blockIdx.x) * kMoveThreads + threadIdx.x; id0 < all;
       id0 += kAhead * step) {
    int32_t to[kAhead], from[kAhead];
    int piece[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t id = id0 + i * step;
      const int m = id < all ? int(id / lanes) : 0;
      piece[i] = int(id % lanes);
      to[i] = id < all ? dst[m] : -1;
      from[i] = src[m];
    }
    u32x4_t x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      // (a move of a missing page reads row 0 and is not stored)
      const uint8_t* cache = piece[i] < chunks ? a.k_cache : a.v_cache;
      x[i] = *reinterpret_cast<const u32x4_t*>(cache + row_at(max(from[i], 0), piece[i]));
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (to[i] < 0 || from[i] < 0) continue;
      uint8_t* cache = piece[i] < chunks ? a.k_cache : a.v_cache;
      *reinterpret_cast<u32x4_t*>(cache + row_at(to[i], piece[i])) = x[i];
      if (piece[i] == 0) a.scores[score_at(a, to[i], h)] = a.scores[score_at(a, from[i], h)];
      if (piece[i] == 1 && a.positions)
        a.positions[score_at(a, to[i], h)] = a.positions[score_at(a, from[i], h)];
    }
  }
}

// A sequence of n tokens has at most min(keep, n - keep) <= n / 2 moves.
int64_t moves_for(int64_t max_len) { return max_len / 2; }

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int64_t kvc_evict_workspace_bytes(int32_t batch, int32_t num_kv_heads,
                                             int32_t max_seq_len) {
  if (batch <= 0 || num_kv_heads <= 0 || max_seq_len <= 0) return 0;
  return int64_t(batch) * num_kv_heads * (1 + 2 * moves_for(max_seq_len)) * 4;
}

extern "C" int kvc_evict_kv(
    void* key_cache, void* value_cache, int64_t num_blocks, int32_t num_kv_heads,
    int32_t head_dim, int32_t block_size, int32_t elem_bytes, int64_t cache_block_stride,
    int64_t cache_token_stride, float* scores, int32_t* positions,
    const int32_t* block_table, int64_t block_table_row_stride, int32_t block_table_width,
    int32_t block_table_rows, const int32_t* seq_ids, const int32_t* seq_lens,
    const int32_t* keep, const int32_t* recent, const int32_t* position_offsets, int32_t batch,
    int32_t max_seq_len, void* workspace, int64_t workspace_bytes, void* stream) {
  KVC_REQUIRE(batch >= 0 && max_seq_len >= 0, KVC_ERR_INVALID_ARG, "negative size");
  KVC_REQUIRE(num_kv_heads > 0 && head_dim > 0 && elem_bytes > 0, KVC_ERR_INVALID_ARG,
              "bad head count, head_dim or element size");
  const int64_t row = int64_t(head_dim) * elem_bytes;
  KVC_REQUIRE(block_size == kPage, KVC_ERR_UNSUPPORTED, "eviction supports block_size 16");
  KVC_REQUIRE(row % 16 == 0 && row <= 65536, KVC_ERR_UNSUPPORTED,
              "a head's row must be a multiple of 16 bytes, at most 64 KiB");
  KVC_REQUIRE(int64_t(batch) * num_kv_heads < 65536, KVC_ERR_UNSUPPORTED,
              "eviction takes fewer than 65536 (sequence, KV head) pairs at once");
  if (batch == 0 || max_seq_len == 0) return ok();
  KVC_REQUIRE(key_cache && value_cache && scores && block_table && seq_lens && keep && recent,
              KVC_ERR_INVALID_ARG, "null pointer");
  KVC_REQUIRE(num_blocks < (int64_t(1) << 27), KVC_ERR_UNSUPPORTED,
              "eviction takes caches of fewer than 2^27 blocks");
  KVC_REQUIRE(aligned(scores, 16) && aligned(positions, 16), KVC_ERR_ALIGNMENT,
              "scores and positions must be 16-byte aligned");
  KVC_REQUIRE(num_blocks > 0 && block_table_width >= 0 && block_table_width < (1 << 26) &&
                  block_table_rows > 0 && block_table_row_stride >= block_table_width,
              KVC_ERR_INVALID_ARG, "bad num_blocks or block table");
  KVC_REQUIRE(cache_token_stride >= int64_t(num_kv_heads) * head_dim &&
                  cache_block_stride >= cache_token_stride * kPage,
              KVC_ERR_INVALID_ARG, "cache strides smaller than the block");
  KVC_REQUIRE(aligned(key_cache, 16) && aligned(value_cache, 16) &&
                  cache_block_stride * elem_bytes % 16 == 0 &&
                  cache_token_stride * elem_bytes % 16 == 0,
              KVC_ERR_ALIGNMENT, "caches must be 16-byte aligned with matching strides");
  const int64_t need = kvc_evict_workspace_bytes(batch, num_kv_heads, max_seq_len);
  KVC_REQUIRE(workspace && workspace_bytes >= need, KVC_ERR_WORKSPACE,
              "workspace too small: need " + std::to_string(need) + " bytes");
  KVC_REQUIRE(aligned(workspace, 4), KVC_ERR_ALIGNMENT, "workspace must be 4-byte aligned");
  EvictArgs a;
  a.k_cache = static_cast<uint8_t*>(key_cache);
  a.v_cache = static_cast<uint8_t*>(value_cache);
  a.num_blocks = num_blocks;
  a.block_bytes = cache_block_stride * elem_bytes;
  a.token_bytes = cache_token_stride * elem_bytes;
  a.row_bytes = int32_t(row);
  a.num_kv_heads = num_kv_heads;
  a.scores = scores;
  a.positions = positions;
  a.table = block_table;
  a.table_stride = block_table_row_stride;
  a.table_width = block_table_width;
  a.table_rows = block_table_rows;
  a.seq_ids = seq_ids;
  a.seq_lens = seq_lens;
  a.keep = keep;
  a.recent = recent;
  a.offsets = position_offsets;
  a.batch = batch;
  a.max_len = max_seq_len;
  a.max_moves = int32_t(moves_for(max_seq_len));
  const int64_t pairs = int64_t(batch) * num_kv_heads;
  a.counts = static_cast<int32_t*>(workspace);
  a.dst = a.counts + pairs;
  a.src = a.dst + pairs * a.max_moves;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid{unsigned(num_kv_heads), unsigned(batch)};
  // Four waves for sequences of up to 2048 tokens, with more of them per CU; sixteen
  // for longer ones; as much LDS as their keys take.  Both launches, hardly any moves, 8
  // heads: 64 x 500 tokens 19 us with four waves, 22 with sixteen; 64 x 8000 32 us with
  // 32 KB of keys, 38 with 128 KB; 16 x 30000 42 us with the keys in LDS, 73 from memory.
  if (max_seq_len <= kShortKeys)
    evict_select_kernel<256, kShortKeys><<<grid, 256, 0, s>>>(a);
  else if (max_seq_len <= kMiddleKeys)
    evict_select_kernel<1024, kMiddleKeys><<<grid, 1024, 0, s>>>(a);
  else if (max_seq_len <= kLongKeys)
    evict_select_kernel<1024, kLongKeys><<<grid, 1024, 0, s>>>(a);
  else
    evict_select_kernel<1024, 0><<<grid, 1024, 0, s>>>(a);
  KVC_LAUNCH_CHECK();
  const int64_t per = (int64_t(a.max_moves) * 2 * (row / 16) + kMoveThreads - 1) / kMoveThreads;
  const int64_t chunks = std::max<int64_t>(1, std::min(per, (kMoveWorkgroups + pairs - 1) / pairs));
  evict_move_kernel<<<dim3(unsigned(chunks), unsigned(pairs)), kMoveThreads, 0, s>>>(a);
  KVC_LAUNCH_CHECK();
  return ok();
}
