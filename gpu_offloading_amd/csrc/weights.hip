// Attention weight that every cached token receives, accumulated per KV head:
//   w[t] = sum over query rows (i, g) that see t of exp(scale q_ig . k_t - lse_ig)
//   scores[t] = w[t] (new tokens) or scores[t] + w[t]
// given the log-sum-exp of the attention over the same keys.  The rows of a KV
// head are its `group` query heads of every query token.
//
// Chunk form (weights_chunk_kernel): half of attention's products, one
// exponential each.  S = Q K^T tiles from v_mfma_f32_32x32x16 (A: lane l = row
// l%32, k = 8(l/32)..+7; B: column l%32, same k; C: acc[4i+j] = row
// 8i+4(l/32)+j, column l%32) with query rows as A and keys as B: a key is a
// column, so all its terms end up in two lanes and a row's masks and sums never
// cross lanes.  A wave keeps its keys' K in registers for the whole unit and
// streams Q past them.
//
// Single-token form (weights_token_kernel): reads K once and is bound by that.
#include "kvc_common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "unit_plan.h"

namespace kvc {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kPage = 16;
constexpr float kLog2e = 1.44269504088896340736f;

struct Bf16 {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16_t mfma32(x8 a, x8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mfma16(x8 a, x8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
struct Fp16 {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16_t mfma32(x8 a, x8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mfma16(x8 a, x8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// What both forms share: the cache, its pages and the scores.
struct WeightsArgs {
  const uint16_t* q;
  int64_t q_stride;                // elements between query tokens
  const float* lse;                // [query tokens][Hq]
  const uint16_t* k_cache;
  int64_t block_stride, token_stride, num_blocks;
  const int32_t* indices;
  int64_t num_indices;
  int32_t num_kv_heads, group;
  float scale_log2;                // sm_scale * log2(e)
  float* scores;                   // [num_blocks][Hkv][16]
  int32_t* positions;              // the same, may be null
  const int32_t* offsets;          // by sequence, may be null
  const int32_t* seq_ids;          // request -> sequence, may be null
};

// A key's block: its page's id, or -1 where the page is missing or out of range.
__device__ __forceinline__ int32_t block_of(const WeightsArgs& a, int64_t page) {
  if (page >= a.num_indices) return -1;
  const int32_t id = a.indices[page];
  return id >= 0 && id < a.num_blocks ? id : -1;
}

__device__ __forceinline__ void store_weight(const WeightsArgs& a, int32_t block, int h, int key,
                                             int b, float w, bool fresh) {
  const int64_t at = (int64_t(block) * a.num_kv_heads + h) * kPage + key % kPage;
  a.scores[at] = fresh ? w : a.scores[at] + w;
  if (fresh && a.positions)
    a.positions[at] = key + (a.offsets ? a.offsets[a.seq_ids ? a.seq_ids[b] : b] : 0);
}

struct ChunkArgs {
  WeightsArgs w;
  const int2* wg_units;            // [workgroups]: (first unit, units)
  const int4* units;               // [units][2]: (KV head, first key, q_len, kv_len),
                                   //   (q offset, page offset, request, first new key)
  int32_t causal;
};

constexpr int kChunkThreads = 256;
constexpr int kWaves = kChunkThreads / 64;
constexpr int kRows = 32;          // query rows per MFMA block
template <int D> constexpr int kKeyBlocks = D == 256 ? 2 : 4;   // 32-key blocks per wave

// kShare: the four waves hold the same keys and take every fourth block of
// rows; else they hold consecutive keys and each takes all the rows.
template <typename T, int D, bool kShare>
__global__ __launch_bounds__(kChunkThreads, 2) void weights_chunk_kernel(ChunkArgs c) {
  constexpr int KB = kKeyBlocks<D>, kSteps = D / 16;
  typedef typename T::x8 x8;
  const WeightsArgs& a = c.w;
  __shared__ float lse_s[kWaves][kRows];
  __shared__ int limit_s[kWaves][kRows];
  __shared__ float part[kShare ? kWaves : 1][32 * KB];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 31, half = lane >> 5;
  const int Hq = a.num_kv_heads * a.group;
  const int step_rows = kShare ? kRows * kWaves : kRows;
  const int step_tok = step_rows / a.group, step_head = step_rows % a.group;

  const int2 span = c.wg_units[blockIdx.x];
  for (int u = span.x; u < span.x + span.y; ++u) {
    const int4 x = c.units[2 * u], y = c.units[2 * u + 1];
    const int h = x.x, q_len = x.z, kv_len = x.w;
    const int key0 = x.y + (kShare ? 0 : wave * 32 * KB);
    if (key0 < kv_len) {     // (the same for all waves where they share keys)
      int32_t block[KB];
      x8 kop[KB][kSteps];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int key = key0 + 32 * kb + r;
        block[kb] = key < kv_len ? block_of(a, int64_t(y.y) + key / kPage) : -1;
        // A key that is not there reads block 0; its column is not stored.
        const uint16_t* kp = a.k_cache + int64_t(max(block[kb], 0)) * a.block_stride +
                             (key % kPage) * a.token_stride + h * D + 8 * half;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks)
          kop[kb][ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(kp + 16 * ks));
      }
      // Rows from the first token that sees key0 on.
      const int ahead = kv_len - q_len;        // keys before the first query token
      const int tok0 = c.causal ? max(0, key0 - ahead) : 0;
      const int rows = max(0, q_len - tok0) * a.group;
      const int row0 = kShare ? wave * kRows : 0;
      int tok = tok0 + (row0 + r) / a.group, head = (row0 + r) % a.group;
      float acc[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) acc[kb] = 0.f;

      for (int rb = row0; rb < rows; rb += step_rows) {
        const bool there = rb + r < rows;
        const int64_t qt = int64_t(y.x) + (there ? tok : q_len - 1);
        const int qh = h * a.group + (there ? head : 0);
        x8 qop[kSteps];
        const uint16_t* qp = a.q + qt * a.q_stride + qh * D + 8 * half;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks)
          qop[ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(qp + 16 * ks));
        const float lse = a.lse[qt * Hq + qh];
        // The last key that this row sees; a row of no key (lse -inf) gives nothing.
        const int limit = !there || lse == -INFINITY ? -1 : c.causal ? ahead + tok : kv_len;
        lse_s[wave][r] = lse * -kLog2e;
        limit_s[wave][r] = limit;
        const bool whole = __builtin_amdgcn_ballot_w64(limit < key0 + 32 * KB - 1) == 0;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        float4 nl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          nl[i] = *reinterpret_cast<const float4*>(&lse_s[wave][8 * i + 4 * half]);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          f32x16_t s;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks) s = T::mfma32(qop[ks], kop[kb][ks], s);
          const int key = key0 + 32 * kb + r;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float n4[4] = {nl[i].x, nl[i].y, nl[i].z, nl[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float p = fast_exp2(fmaf(s[4 * i + j], a.scale_log2, n4[j]));
              acc[kb] += whole || key <= limit_s[wave][8 * i + 4 * half + j] ? p : 0.f;
            }
          }
        }
        __builtin_amdgcn_wave_barrier();
        tok += step_tok;
        head += step_head;
        if (head >= a.group) {
          head -= a.group;
          ++tok;
        }
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) acc[kb] += __shfl_xor(acc[kb], 32);
      if (kShare) {
        if (half == 0)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) part[wave][32 * kb + r] = acc[kb];
        __syncthreads();
        const int i = threadIdx.x;
        const int key = key0 + i;
        if (i < 32 * KB && key < kv_len) {
          const float w = (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
          const int32_t blk = block_of(a, int64_t(y.y) + key / kPage);
          if (blk >= 0) store_weight(a, blk, h, key, y.z, w, key >= y.w);
        }
        __syncthreads();
      } else if (half == 0) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int key = key0 + 32 * kb + r;
          if (block[kb] >= 0) store_weight(a, block[kb], h, key, y.z, acc[kb], key >= y.w);
        }
      }
    }
  }
}

struct TokenArgs {
  WeightsArgs w;
  const int32_t* indptr;           // [batch + 1] pages
  const int32_t* last_page_len;
  int32_t batch;
};

constexpr int kTokenPages = 4;     // pages of one head per wave and step
constexpr int kTokenThreads = 256;
constexpr int64_t kTokenWorkgroups = 4096;   // at most; waves take further tasks in turn

// A wave takes kTokenPages consecutive entries of the batch's page list for one
// KV head (heads fastest: neighbouring waves read the same tokens' rows).  S =
// Q K^T per page with v_mfma_f32_16x16x32 (A: lane l = row l%16, k = 8(l/16)..+7;
// B: column l%16; C: acc[j] = row 4(l/16)+j, column l%16): rows are the group's
// query heads, columns the page's tokens.
template <typename T, int D>
__global__ __launch_bounds__(kTokenThreads) void weights_token_kernel(TokenArgs c) {
  constexpr int kSteps = D / 32;
  typedef typename T::x8 x8;
  const WeightsArgs& a = c.w;
  const int lane = threadIdx.x & 63, r = lane & 15, quad = lane >> 4;
  const int Hq = a.num_kv_heads * a.group;
  const int64_t pages = min(int64_t(c.indptr[c.batch]), a.num_indices);
  const int64_t tasks = (pages + kTokenPages - 1) / kTokenPages * a.num_kv_heads;
  const int64_t waves = int64_t(gridDim.x) * (kTokenThreads / 64);
  for (int64_t task = int64_t(blockIdx.x) * (kTokenThreads / 64) +
                      __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
       task < tasks; task += waves) {
    const int h = int(task % a.num_kv_heads);
    const int64_t p0 = task / a.num_kv_heads * kTokenPages;
    int32_t block[kTokenPages];
    x8 kop[kTokenPages][kSteps];
#pragma unroll
    for (int i = 0; i < kTokenPages; ++i) {
      block[i] = p0 + i < pages ? __builtin_amdgcn_readfirstlane(block_of(a, p0 + i)) : -1;
      const uint16_t* kp = a.k_cache + int64_t(max(block[i], 0)) * a.block_stride +
                           r * a.token_stride + h * D + 8 * quad;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
        kop[i][ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(kp + 32 * ks));
    }
#pragma unroll
    for (int i = 0; i < kTokenPages; ++i) {
      if (block[i] < 0) continue;
      // The request: the last one whose pages start at or before this one.
      const int64_t p = p0 + i;
      int b = 0;
      for (int base = 0; base < c.batch; base += 64) {
        const int at = base + lane;
        const bool before = at < c.batch && c.indptr[at + 1] <= p;
        b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
      }
      if (b >= c.batch) continue;
      const int first = c.indptr[b], last = c.indptr[b + 1] - 1;
      const int tokens = p < last ? kPage : c.last_page_len[b];
      float w = 0.f;
      for (int g0 = 0; g0 < a.group; g0 += 16) {
        const int n = min(16, a.group - g0);
        const int64_t qh = int64_t(h) * a.group + g0 + min(r, n - 1);
        const uint16_t* qp = a.q + b * a.q_stride + qh * D + 8 * quad;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks)
          s = T::mfma16(__builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(qp + 32 * ks)),
                        kop[i][ks], s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 4 * quad + j;
          const float lse = a.lse[int64_t(b) * Hq + h * a.group + g0 + min(row, n - 1)];
          const float e = fast_exp2(fmaf(s[j], a.scale_log2, lse * -kLog2e));
          w += row < n && lse != -INFINITY ? e : 0.f;
        }
      }
      w += __shfl_xor(w, 16);
      w += __shfl_xor(w, 32);
      const int key = int(p - first) * kPage + r;
      if (quad == 0 && r < tokens)
        store_weight(a, block[i], h, key, b, w, p == last && r == tokens - 1);
    }
  }
}

constexpr int64_t kMaxWorkgroups = 512;
constexpr int kShareBlocks = 16;   // row blocks of a request from which waves share keys
int64_t plan_workgroups(int64_t units) { return std::min(kMaxWorkgroups, units); }
int unit_keys(int head_dim, int share) {
  return 32 * (head_dim == 256 ? 2 : 4) * (share ? 1 : kWaves);
}
constexpr int kMaxGroup = 128;

int weights_plan(const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* lpl,
                 const int32_t* new_tokens, int32_t batch, int32_t hq, int32_t hkv,
                 int32_t head_dim, int32_t page_size, int32_t causal,
                 kvc_weights_schedule* sched, int32_t* plan_host, int64_t plan_capacity) {
  KVC_REQUIRE(sched, KVC_ERR_INVALID_ARG, "null schedule");
  KVC_REQUIRE(batch >= 0, KVC_ERR_INVALID_ARG, "negative batch");
  KVC_REQUIRE(batch == 0 || (qo_indptr && kv_indptr && lpl), KVC_ERR_INVALID_ARG,
              "null indptr / last_page_len");
  KVC_REQUIRE(hkv > 0 && hq > 0 && hq % hkv == 0, KVC_ERR_INVALID_ARG,
              "num_qo_heads must be a positive multiple of num_kv_heads");
  const int group = hq / hkv;
  KVC_REQUIRE((head_dim == 64 || head_dim == 128 || head_dim == 256) && page_size == kPage &&
                  group <= kMaxGroup,
              KVC_ERR_UNSUPPORTED, "attention weights support head_dim 64, 128, 256, page_size "
                                   "16 and groups up to 128");
  int64_t most = 0, n = 0, total_kv = 0;
  for (int b = 0; b < batch; ++b) {
    const int64_t q_len = int64_t(qo_indptr[b + 1]) - qo_indptr[b];
    const int64_t pages = int64_t(kv_indptr[b + 1]) - kv_indptr[b];
    KVC_REQUIRE(q_len >= 0 && pages >= 0 && qo_indptr[b] >= 0 && kv_indptr[b] >= 0,
                KVC_ERR_INVALID_ARG, "qo_indptr and kv_indptr must be non-negative and "
                                     "non-decreasing");
    KVC_REQUIRE(pages == 0 || (lpl[b] >= 1 && lpl[b] <= kPage), KVC_ERR_INVALID_ARG,
                "last_page_len must be in 1..page_size for a request with pages");
    const int64_t kv_len = pages > 0 ? (pages - 1) * kPage + lpl[b] : 0;
    KVC_REQUIRE(kv_len < (int64_t(1) << 30), KVC_ERR_INVALID_ARG, "request too long");
    KVC_REQUIRE(q_len <= kv_len && q_len * group < (int64_t(1) << 30), KVC_ERR_INVALID_ARG,
                "queries must be a request's last cached tokens");
    KVC_REQUIRE(!new_tokens || (new_tokens[b] >= 0 && new_tokens[b] <= kv_len),
                KVC_ERR_INVALID_ARG, "new_tokens outside the request");
    most = std::max(most, (q_len * group + kRows - 1) / kRows);
    total_kv += kv_len;
  }
  const int share = most >= kShareBlocks;
  const int keys = unit_keys(head_dim, share);
  KVC_REQUIRE((total_kv / keys + batch) * hkv < (int64_t(1) << 27), KVC_ERR_INVALID_ARG,
              "too many (key tile, KV head) units");
  std::vector<int32_t> rec;
  for (int b = 0; b < batch; ++b) {
    const int q_len = qo_indptr[b + 1] - qo_indptr[b];
    const int pages = kv_indptr[b + 1] - kv_indptr[b];
    const int kv_len = pages > 0 ? (pages - 1) * kPage + lpl[b] : 0;
    const int nnew = new_tokens ? new_tokens[b] : q_len;
    if (q_len == 0 && nnew == 0) continue;
    // Without queries only the new tokens change (to 0).
    for (int k0 = q_len ? 0 : (kv_len - nnew) / keys * keys; k0 < kv_len; k0 += keys) {
      const int64_t t0 = causal ? std::max(0, k0 - (kv_len - q_len)) : 0;
      const int64_t blocks = (std::max<int64_t>(0, q_len - t0) * group + kRows - 1) / kRows;
      const int32_t r8[kUnitInts] = {b, k0, q_len, kv_len, qo_indptr[b], kv_indptr[b],
                                     int32_t(blocks), kv_len - nnew};
      rec.insert(rec.end(), r8, r8 + kUnitInts);
      ++n;
    }
  }
  const int64_t W = plan_workgroups(n * hkv);
  sched->batch = batch;
  sched->num_qo_heads = hq;
  sched->num_kv_heads = hkv;
  sched->head_dim = head_dim;
  sched->page_size = page_size;
  sched->causal = causal ? 1 : 0;
  sched->shared_keys = share;
  sched->num_units = int32_t(n * hkv);
  sched->num_workgroups = int32_t(W);
  sched->total_q = batch ? qo_indptr[batch] : 0;
  sched->plan_ints = unit_table_ints(W) + n * hkv * kUnitInts;
  KVC_REQUIRE(plan_capacity >= sched->plan_ints && (plan_host || sched->plan_ints == 0),
              KVC_ERR_WORKSPACE,
              "plan buffer too small: need " + std::to_string(sched->plan_ints) + " int32");
  write_unit_plan(rec, n, hkv, W, plan_host);
  // Entry 6, the planner's cost, becomes the request (a unit has keys, so it is the
  // last one whose pages start at the unit's).
  int32_t* units = plan_host + unit_table_ints(W);
  for (int64_t u = 0; u < n * hkv; ++u) {
    const int32_t off = units[u * kUnitInts + 5];
    const int32_t* p = std::upper_bound(kv_indptr, kv_indptr + batch, off);
    units[u * kUnitInts + 6] = int32_t(p - kv_indptr) - 1;
  }
  return ok();
}

int check_common(const WeightsArgs& a, int Hq, int Hkv, int D, const char* who) {
  KVC_REQUIRE(a.k_cache && a.scores && a.indices, KVC_ERR_INVALID_ARG,
              std::string(who) + ": null pointer");
  KVC_REQUIRE(a.num_blocks > 0 && a.num_indices > 0, KVC_ERR_INVALID_ARG,
              std::string(who) + ": bad num_blocks or empty indices");
  KVC_REQUIRE(a.token_stride >= int64_t(Hkv) * D && a.block_stride >= a.token_stride * kPage,
              KVC_ERR_INVALID_ARG, std::string(who) + ": cache strides smaller than the block");
  KVC_REQUIRE(a.q_stride >= int64_t(Hq) * D, KVC_ERR_INVALID_ARG,
              std::string(who) + ": q token stride smaller than Hq*head_dim");
  KVC_REQUIRE(aligned(a.q, 16) && aligned(a.k_cache, 16) && a.q_stride % 8 == 0 &&
                  a.block_stride % 8 == 0 && a.token_stride % 8 == 0,
              KVC_ERR_ALIGNMENT,
              std::string(who) + ": q and the cache must be 16-byte aligned with strides that "
                                 "are multiples of 8");
  return ok();
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_weights_plan(const int32_t* qo_indptr_host, const int32_t* kv_indptr_host,
                                const int32_t* last_page_len_host,
                                const int32_t* new_tokens_host, int32_t batch,
                                int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                int32_t page_size, int32_t causal,
                                kvc_weights_schedule* schedule, int32_t* plan_host,
                                int64_t plan_capacity) {
  KVC_NO_THROW(return weights_plan(qo_indptr_host, kv_indptr_host, last_page_len_host,
                                   new_tokens_host, batch, num_qo_heads, num_kv_heads, head_dim,
                                   page_size, causal, schedule, plan_host, plan_capacity));
}

extern "C" int kvc_batch_attention_weights_run(
    const kvc_weights_schedule* sched, const int32_t* plan, const void* q,
    int64_t q_token_stride, const float* lse, const void* key_cache,
    int64_t cache_block_stride, int64_t cache_token_stride, int64_t num_blocks,
    const int32_t* indices, int64_t num_indices, int32_t dtype, float sm_scale, float* scores,
    int32_t* positions, const int32_t* position_offsets, const int32_t* seq_ids, void* stream) {
  KVC_REQUIRE(sched, KVC_ERR_INVALID_ARG, "null schedule");
  const int Hq = sched->num_qo_heads, Hkv = sched->num_kv_heads, D = sched->head_dim;
  KVC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= kMaxGroup &&
                  (D == 64 || D == 128 || D == 256) && sched->page_size == kPage &&
                  sched->num_units >= 0 &&
                  sched->num_workgroups == plan_workgroups(sched->num_units) &&
                  sched->plan_ints == unit_table_ints(sched->num_workgroups) +
                                          int64_t(sched->num_units) * kUnitInts,
              KVC_ERR_INVALID_ARG, "schedule not produced by kvc_weights_plan");
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");
  KVC_REQUIRE(std::isfinite(sm_scale), KVC_ERR_INVALID_ARG, "sm_scale must be finite");
  if (sched->num_units == 0) return ok();
  KVC_REQUIRE(plan && (sched->total_q == 0 || (q && lse)), KVC_ERR_INVALID_ARG, "null pointer");
  KVC_REQUIRE(aligned(plan, 16), KVC_ERR_ALIGNMENT, "plan must be 16-byte aligned");
  ChunkArgs c;
  c.w = WeightsArgs{static_cast<const uint16_t*>(q), q_token_stride, lse,
                    static_cast<const uint16_t*>(key_cache), cache_block_stride,
                    cache_token_stride, num_blocks, indices, num_indices, Hkv, Hq / Hkv,
                    sm_scale * kLog2e, scores, positions, position_offsets, seq_ids};
  if (const int st = check_common(c.w, Hq, Hkv, D, "kvc_batch_attention_weights_run")) return st;
  c.wg_units = reinterpret_cast<const int2*>(plan);
  c.units = reinterpret_cast<const int4*>(plan + unit_table_ints(sched->num_workgroups));
  c.causal = sched->causal;
  const dim3 grid(static_cast<unsigned>(sched->num_workgroups));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto t, auto share) {
    typedef decltype(t) T;
    constexpr bool kS = decltype(share)::value;
    if (D == 64) weights_chunk_kernel<T, 64, kS><<<grid, kChunkThreads, 0, s>>>(c);
    else if (D == 128) weights_chunk_kernel<T, 128, kS><<<grid, kChunkThreads, 0, s>>>(c);
    else weights_chunk_kernel<T, 256, kS><<<grid, kChunkThreads, 0, s>>>(c);
  };
  if (dtype == KVC_DTYPE_BF16) {
    if (sched->shared_keys) launch(Bf16{}, std::true_type{});
    else launch(Bf16{}, std::false_type{});
  } else {
    if (sched->shared_keys) launch(Fp16{}, std::true_type{});
    else launch(Fp16{}, std::false_type{});
  }
  KVC_LAUNCH_CHECK();
  return ok();
}

extern "C" int kvc_decode_attention_weights(
    const void* q, int64_t q_token_stride, const float* lse, const void* key_cache,
    int64_t cache_block_stride, int64_t cache_token_stride, int64_t num_blocks,
    const int32_t* indptr, const int32_t* indices, int64_t num_indices,
    const int32_t* last_page_len, int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t page_size, int32_t dtype, float sm_scale, float* scores,
    int32_t* positions, const int32_t* position_offsets, const int32_t* seq_ids, void* stream) {
  const int Hq = num_qo_heads, Hkv = num_kv_heads, D = head_dim;
  KVC_REQUIRE(batch >= 0, KVC_ERR_INVALID_ARG, "negative batch");
  KVC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, KVC_ERR_INVALID_ARG,
              "num_qo_heads must be a positive multiple of num_kv_heads");
  KVC_REQUIRE((D == 64 || D == 128 || D == 256) && page_size == kPage && Hq / Hkv <= kMaxGroup,
              KVC_ERR_UNSUPPORTED, "attention weights support head_dim 64, 128, 256, page_size "
                                   "16 and groups up to 128");
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");
  KVC_REQUIRE(std::isfinite(sm_scale), KVC_ERR_INVALID_ARG, "sm_scale must be finite");
  if (batch == 0 || num_indices == 0) return ok();
  KVC_REQUIRE(q && lse && indptr && last_page_len, KVC_ERR_INVALID_ARG, "null pointer");
  TokenArgs c;
  c.w = WeightsArgs{static_cast<const uint16_t*>(q), q_token_stride, lse,
                    static_cast<const uint16_t*>(key_cache), cache_block_stride,
                    cache_token_stride, num_blocks, indices, num_indices, Hkv, Hq / Hkv,
                    sm_scale * kLog2e, scores, positions, position_offsets, seq_ids};
  if (const int st = check_common(c.w, Hq, Hkv, D, "kvc_decode_attention_weights")) return st;
  c.indptr = indptr;
  c.last_page_len = last_page_len;
  c.batch = batch;
  const int64_t tasks = (num_indices + kTokenPages - 1) / kTokenPages * Hkv;
  const int64_t wgs = (tasks + kTokenThreads / 64 - 1) / (kTokenThreads / 64);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(wgs, kTokenWorkgroups)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto t) {
    typedef decltype(t) T;
    if (D == 64) weights_token_kernel<T, 64><<<grid, kTokenThreads, 0, s>>>(c);
    else if (D == 128) weights_token_kernel<T, 128><<<grid, kTokenThreads, 0, s>>>(c);
    else weights_token_kernel<T, 256><<<grid, kTokenThreads, 0, s>>>(c);
  };
  if (dtype == KVC_DTYPE_BF16) launch(Bf16{});
  else launch(Fp16{});
  KVC_LAUNCH_CHECK();
  return ok();
}
