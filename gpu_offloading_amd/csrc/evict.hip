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
// writes the move list.  evict_move_kernel: K, V, score and position of each move.
#include "kvc_common.h"

#include <algorithm>

namespace kvc {
namespace {

constexpr int kPage = 16;
constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 256;
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
  int32_t* dst;                                   // [batch][Hkv][max_moves] slots
  int32_t* src;
};

__device__ __forceinline__ const int32_t* table_row(const EvictArgs& a, int b) {
  const int row = a.seq_ids ? a.seq_ids[b] : b;
  return row >= 0 && row < a.table_rows ? a.table + row * a.table_stride : nullptr;
}

// Index of (slot, head) in the scores, or -1 where the slot's page is missing.
__device__ __forceinline__ int64_t score_at(const EvictArgs& a, const int32_t* row, int slot,
                                            int h) {
  const int32_t id = row[slot / kPage];
  return id >= 0 && id < a.num_blocks
             ? (int64_t(id) * a.num_kv_heads + h) * kPage + slot % kPage : -1;
}

// Scores as unsigned keys of the same order; -0 is 0, every NaN ranks above inf.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) return kNanKey;
  const uint32_t u = __float_as_uint(s + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of v over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int2 block_scan(int v, int* wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) wave_sums[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    before += w < wave ? wave_sums[w] : 0;
    all += wave_sums[w];
  }
  return make_int2(before + x - v, all);
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[kBins];
  __shared__ int wave_sums[kSelectWaves];
  __shared__ int found[2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int32_t* row = table_row(a, b);
  const int n = row ? min(min(a.seq_lens[b], a.max_len), a.table_width * kPage) : 0;
  const int keep = min(max(a.keep[b], 0), n);
  int* count = a.counts + int64_t(b) * a.num_kv_heads + h;
  if (n <= keep) {
    if (threadIdx.x == 0) *count = 0;
    return;
  }
  const int offset = a.positions && a.offsets ? a.offsets[b] : 0;
  const int64_t recent_from = int64_t(n) + offset - max(a.recent[b], 0);
  auto key_of = [&](int slot) __attribute__((always_inline)) -> uint32_t {
    const int64_t at = score_at(a, row, slot, h);
    if (at < 0) return 0u;   // ranks last
    const int64_t place = a.positions ? a.positions[at] : slot;
    return place >= recent_from ? kRecentKey : score_key(a.scores[at]);
  };

  // Radix select of the keep-th largest key, 8 bits at a time: `prefix` holds
  // the key's bits found so far, `want` how many keys with that prefix stay.
  uint32_t prefix = 0;
  int want = keep;
  for (int shift = 24; want > 0 && shift >= 0; shift -= 8) {
    if (threadIdx.x < kBins) hist[threadIdx.x] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < n; s += kSelectThreads) {
      const uint32_t k = key_of(s);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // Keys in larger bins than this thread's: bins are scanned from the top.
    const int bin = kBins - 1 - int(threadIdx.x);
    const int c = threadIdx.x < kBins ? hist[bin] : 0;
    const int above = block_scan(c, wave_sums).x;
    if (threadIdx.x < kBins && above < want && want <= above + c) {
      found[0] = bin;
      found[1] = want - above;
    }
    __syncthreads();
    prefix |= uint32_t(found[0]) << shift;
    want = found[1];
  }
  // Keys above `prefix` stay, and the first `want` equal to it by slot.
  int ties = 0, holes = 0, sources = 0;   // found so far, over the workgroup
  int32_t* dst = a.dst + (int64_t(b) * a.num_kv_heads + h) * a.max_moves;
  int32_t* src = a.src + (int64_t(b) * a.num_kv_heads + h) * a.max_moves;
  for (int base = 0; base < n; base += kSelectThreads) {
    const int s = base + threadIdx.x;
    const uint32_t k = s < n ? key_of(s) : 0u;
    const bool tie = keep > 0 && s < n && k == prefix;
    const int2 t = block_scan(tie, wave_sums);
    const bool stays = keep > 0 && s < n && (k > prefix || (tie && ties + t.x < want));
    ties += t.y;
    const bool hole = s < keep && !stays, source = s >= keep && stays;
    const int2 m = block_scan(hole | (source << 16), wave_sums);
    if (hole) {
      const int i = holes + (m.x & 0xffff);
      if (i < a.max_moves) dst[i] = s;
    }
    if (source) {
      const int i = sources + (m.x >> 16);
      if (i < a.max_moves) src[i] = s;
    }
    holes += m.y & 0xffff;
    sources += m.y >> 16;
  }
  if (threadIdx.x == 0) *count = min(holes, a.max_moves);
}

constexpr int kMoveThreads = 256;

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  const int h = blockIdx.y % a.num_kv_heads, b = blockIdx.y / a.num_kv_heads;
  const int64_t list = int64_t(b) * a.num_kv_heads + h;
  const int32_t* row = table_row(a, b);
  const int count = a.counts[list];
  const int chunks = a.row_bytes / 16;             // 16-byte pieces of a row
  const int lanes = 2 * chunks;                    // K's pieces, then V's
  for (int64_t id = int64_t(blockIdx.x) * kMoveThreads + threadIdx.x;
       id < int64_t(count) * lanes; id += int64_t(gridDim.x) * kMoveThreads) {
    const int i = int(id / lanes), c = int(id % lanes);
    const int d = a.dst[list * a.max_moves + i], s = a.src[list * a.max_moves + i];
    const int64_t db = row[d / kPage], sb = row[s / kPage];
    if (db < 0 || db >= a.num_blocks || sb < 0 || sb >= a.num_blocks) continue;
    uint8_t* cache = c < chunks ? a.k_cache : a.v_cache;
    const int64_t in = int64_t(h) * a.row_bytes + (c % chunks) * 16;
    *reinterpret_cast<uint4*>(cache + db * a.block_bytes + (d % kPage) * a.token_bytes + in) =
        *reinterpret_cast<const uint4*>(cache + sb * a.block_bytes +
                                        (s % kPage) * a.token_bytes + in);
    if (c == 0) {
      const int64_t to = (db * a.num_kv_heads + h) * kPage + d % kPage;
      const int64_t from = (sb * a.num_kv_heads + h) * kPage + s % kPage;
      a.scores[to] = a.scores[from];
      if (a.positions) a.positions[to] = a.positions[from];
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
  evict_select_kernel<<<dim3(unsigned(num_kv_heads), unsigned(batch)), kSelectThreads, 0, s>>>(a);
  KVC_LAUNCH_CHECK();
  const int64_t per = (int64_t(a.max_moves) * 2 * (row / 16) + kMoveThreads - 1) / kMoveThreads;
  const int64_t chunks = std::max<int64_t>(1, std::min(per, (4096 + pairs - 1) / pairs));
  evict_move_kernel<<<dim3(unsigned(chunks), unsigned(pairs)), kMoveThreads, 0, s>>>(a);
  KVC_LAUNCH_CHECK();
  return ok();
}
