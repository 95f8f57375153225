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
// column, so all its terms end up in two lanes (fp32 sums in row order, joined at the
// end) and a row's masks and sums never cross lanes.  A wave keeps its keys' K in registers for the whole unit and
// streams Q past them.
//
// Single-token form (weights_token_kernel): reads K once and is bound by that.
#include "kvc_common.h"
#include "weights_rows.h"

#include <algorithm>
#include <array>
#include <cmath>
#include <functional>
#include <type_traits>
#include <vector>

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
  const int32_t* offsets;          // [num_offsets] by sequence, may be null
  int32_t num_offsets;
  const int32_t* seq_ids;          // request -> sequence, may be null
};

// A key's block: its page's id, or -1 where the page is missing or out of range.
__device__ __forceinline__ int32_t block_of(const WeightsArgs& a, int64_t page) {
  const int32_t id = a.indices[min(page, a.num_indices - 1)];
  return page < a.num_indices && id >= 0 && id < a.num_blocks ? id : -1;
}

// The position of a request's first cached token (0 where its sequence has no entry).
__device__ __forceinline__ int32_t first_position(const WeightsArgs& a, int b) {
  if (!a.offsets) return 0;
  const int32_t seq = a.seq_ids ? a.seq_ids[b] : b;
  return seq >= 0 && seq < a.num_offsets ? a.offsets[seq] : 0;
}

__device__ __forceinline__ void store_weight(const WeightsArgs& a, int32_t block, int h, int key,
                                             int b, float w, bool fresh) {
  const int64_t at = (int64_t(block) * a.num_kv_heads + h) * kPage + key % kPage;
  a.scores[at] = fresh ? w : a.scores[at] + w;
  if (fresh && a.positions) a.positions[at] = key + first_position(a, b);
}

// A work unit: kUnitKeys keys of one request and KV head, against a run of the
// row blocks that see them.  Record (kRecInts int32):
//   KV head, first key, q_len, kv_len | q offset, page offset, request, first new key |
//   first block, blocks, partial (-1: the unit's sums are the keys' weights), next
// Workgroup w begins with unit w and goes on with the next ones (0: none).
constexpr int kRecInts = 12;
constexpr int kJoinInts = 8;
constexpr int kKeyBlocks = 2;                      // 32-key blocks per wave
constexpr int kWaveKeys = 32 * kKeyBlocks;
constexpr int kChunkThreads = 256;
constexpr int kUnitKeys = kChunkThreads / 64 * kWaveKeys;
constexpr int kWaitLoads = 0x0f70;                 // s_waitcnt vmcnt(0)

struct ChunkArgs {
  WeightsArgs w;
  const int4* units;               // [units][3]
  float* parts;                    // [partials][kUnitKeys]
  int32_t causal;
};

typedef __attribute__((address_space(3))) void lds_void_t;

// The first query token of a unit (causal: the first that sees one of its keys).
__host__ __device__ inline int first_token(int key0, int q_len, int kv_len, int causal) {
  const int t = key0 - (kv_len - q_len);
  return causal && t > 0 ? t : 0;
}

// A workgroup's four waves hold kWaveKeys keys of its unit each, K in registers for
// the whole unit (B operands), and walk the same rows, which arrive in LDS a stage of
// two blocks ahead (global_load_lds, each wave a quarter).  Per 32 rows x 64 keys a
// wave issues, at head_dim 128, 16 matrix instructions of 32 cycles, 32 exponentials of
// 8 and 64 other vector instructions of 4, so in the walk the vector unit is the bound
// (about 600 cycles; a block takes 800); three waves per SIMD share it, one's products
// beside the others' exponentials.  Units of few rows are bound by their start: K is
// waited for before the first product.  Masks are a comparison per weight with the first row that sees the
// lane's key; with that instead of each row's limit read across lanes, and priorities
// that go round, 4 prompts of 2000 tokens went from 93 to 83 us.
// Measured (bf16, head_dim 128, 32 / 8 heads): 2000 rows against 16000 keys 245 to 250
// us (1005 to 985 TFLOP/s), 4 prompts of 1200 to 2048 tokens 64 us (the walk is half of
// it), 8 windows of 32 against 4096 22 us.  Products of the next block interleaved with the exponentials in one wave,
// at two waves per SIMD, took 10% longer.
template <typename T, int D>
__global__ __launch_bounds__(kChunkThreads, D == 64 ? 4 : D == 128 ? 3 : 2)
void weights_chunk_kernel(ChunkArgs c) {
  constexpr int KB = kKeyBlocks, kSteps = D / 16, kRow = 2 * D, kChunks = kRow / 16;
  constexpr int kDma = kStage * kRow / 1024 / 4;   // row loads per wave and stage
  constexpr int kLoadRows = 1024 / kRow;           // rows per load
  constexpr int kAhead = 3;                        // Q operands read ahead
  typedef typename T::x8 x8;
  const WeightsArgs& a = c.w;
  __shared__ struct alignas(16) {
    uint8_t q[2][kStage * kRow];                   // 16-byte chunks XOR-swizzled by row
    float lse[2][4][kStage];                       // each wave's own copy
    float shift[4][kStage];                        // -log2(e) lse of the current stage
  } lds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 31, half = lane >> 5;
  const int Hq = a.num_kv_heads * a.group;
  auto rfl = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  auto lds_addr = [](const void* p) __attribute__((always_inline)) {
    return __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void_t*)p)));
  };
  const uint32_t q_base = lds_addr(lds.q[0] + wave * kDma * 1024);
  const uint32_t lse_base = lds_addr(lds.lse[0][wave]);
  const uint32_t recip = rfl((65536 + a.group - 1) / a.group);   // row / group for row < 192
  auto split = [&](int row, int& tok, int& head) __attribute__((always_inline)) {
    tok = __umul24(row, recip) >> 16;
    head = row - __umul24(tok, a.group);
  };
  const uint32_t q_bytes = uint32_t(a.q_stride * 2);

  // Of a SIMD's waves the hardware prefers the oldest: with equal work the youngest
  // ends last, alone.  Priorities that go round by stage let each be preferred in turn.
  int turn = blockIdx.x / 256 % 3;
  int u = blockIdx.x;
  do {
    const int4 x = c.units[3 * u], y = c.units[3 * u + 1], z = c.units[3 * u + 2];
    const int h = rfl(x.x), key_first = rfl(x.y), q_len = rfl(x.z), kv_len = rfl(x.w);
    const int first_block = rfl(z.x), blocks = rfl(z.y);
    const int stages = (blocks + 1) / 2;
    const int key0 = key_first + wave * kWaveKeys;
    const int ahead = kv_len - q_len;              // keys before the first query token
    const int tok0 = first_token(key_first, q_len, kv_len, c.causal);
    const int last_tok = q_len - 1 - tok0;

    // The stage that is loaded next, tokens from tok0 on, and the bases of its first
    // row's token.  The rows' 32-bit offsets from them are the same in every stage
    // where the group divides 64 and no token ends.
    RowWalk at(a.group, last_tok, first_block * kRows);
    const int step_tok = at.step_tok, step_head = at.step_head;
    int my_base = at.tok, my_first = at.head;      // of the stage being computed
    const uint8_t* st_q = reinterpret_cast<const uint8_t*>(
        a.q + (int64_t(y.x) + tok0 + at.tok) * a.q_stride + h * a.group * D);
    const uint8_t* st_lse = reinterpret_cast<const uint8_t*>(
        a.lse + (int64_t(y.x) + tok0 + at.tok) * Hq + h * a.group);
    uint32_t q_off[kDma], lse_off;
    auto offsets = [&]() __attribute__((always_inline)) {
      const int left = at.left();
      int tok, head;
#pragma unroll
      for (int i = 0; i < kDma; ++i) {
        const int row = (wave * kDma + i) * kLoadRows + lane / kChunks;
        const int chunk = (lane % kChunks) ^ (D == 64 ? (row >> 1) & 7 : row & 15);
        split(at.head + row, tok, head);
        q_off[i] = uint32_t(min(tok, left)) * q_bytes + head * kRow + chunk * 16;
      }
      split(at.head + lane, tok, head);
      lse_off = (uint32_t(min(tok, left)) * Hq + head) * 4;
    };
    // Load i of a stage's kDma + 1 into `slot` (inline assembly: the compiler would wait
    // for all of them at every LDS read; it uses M0 nowhere itself).
    auto stage_load = [&](int i, int slot) __attribute__((always_inline)) {
      if (i < kDma)
        asm volatile(KVC_SET_M0("%0") "global_load_lds_dwordx4 %1, %2"
                     :: "s"(q_base + uint32_t(slot * kStage * kRow + i * 1024)), "v"(q_off[i]),
                        "s"(st_q) : "memory");
      else
        asm volatile(KVC_SET_M0("%0") "global_load_lds_dword %1, %2"
                     :: "s"(lse_base + uint32_t(slot * 4 * kStage * 4)), "v"(lse_off), "s"(st_lse)
                     : "memory");
    };
    // Behind the last stage the last one is loaded again, which nothing reads.
    auto stage_prepare = [&]() __attribute__((always_inline)) {
      const uint32_t tok = uint32_t(at.next());
      st_q += tok * q_bytes;                       // (64 of less than 2^26 bytes at most)
      st_lse += tok * uint32_t(Hq * 4);
      if (at.offsets_change()) offsets();
    };
    offsets();
    if (stages > 0) {
#pragma unroll
      for (int i = 0; i <= kDma; ++i) stage_load(i, 0);
      stage_prepare();
    }

    x8 kop[KB][kSteps];
    int32_t block[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int key = min(key0 + 32 * kb + r, kv_len - 1);
      block[kb] = block_of(a, int64_t(y.y) + key / kPage);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      // A page that is not there reads block 0; its columns are not stored.
      const uint16_t* kp = a.k_cache + int64_t(max(block[kb], 0)) * a.block_stride +
                           (r % kPage) * a.token_stride + h * D + 8 * half;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
        kop[kb][ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(kp + 16 * ks));
    }
    // K and the first stage are here before the walk (waits for K inside it would wait
    // for the rows in flight).
    __builtin_amdgcn_s_waitcnt(kWaitLoads);
    __syncthreads();
    float acc[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) acc[kb] = 0.f;

    // Whether a row of block n of stage st does not see all of the wave's keys.
    auto partly = [&](int n) __attribute__((always_inline)) {
      const int tok = my_base + int(((my_first + kRows * n) * recip) >> 16);
      return c.causal && ahead + tok0 + tok < key0 + kWaveKeys - 1;
    };
    // The first row that sees the lane's key (row 0 is the unit's).
    int sees[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      sees[kb] = !c.causal ? 0 : max(key0 + 32 * kb + r - ahead - tok0, 0) * a.group -
                                     first_block * kRows;
    auto advance = [&]() __attribute__((always_inline)) {
      my_base += step_tok;
      my_first += step_head;
      if (my_first >= a.group) {
        my_first -= a.group;
        ++my_base;
      }
    };
    // The lane's first Q operand of a block, in the current slot.
    uint32_t q_at = r * kRow + (half ^ (D == 64 ? (r >> 1) & 7 : r & 15)) * 16;
    f32x16_t zero, sc[KB];
#pragma unroll
    for (int e = 0; e < 16; ++e) zero[e] = 0.f;
    // Scores of block n of the current slot, `step` behind each step's instructions.
    auto scores = [&](int n, auto step) __attribute__((always_inline)) {
      x8 qop[kSteps];
      uint32_t at = q_at;
      asm volatile("" : "+v"(at));                 // (or every step's place stays in a register)
      auto read_q = [&](int ks) __attribute__((always_inline)) {
        qop[ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(
            lds.q[0] + n * kRows * kRow + (at ^ (32 * ks))));
      };
#pragma unroll
      for (int ks = 0; ks < kAhead; ++ks) read_q(ks);
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) {
        if (ks + kAhead < kSteps) read_q(ks + kAhead);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          sc[kb] = T::mfma32(qop[ks], kop[kb][ks], ks == 0 ? zero : sc[kb]);
        step(ks);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // And their exponentials: accumulator entry 4i+j is row 8i + 4half + j, the lane's
    // column key r.  kMask 1: rows in front of a key's first one do not see it; 2: and
    // rows of lse -inf, whatever their products are, give nothing.
    auto exps = [&](auto kMask, int st, int n) __attribute__((always_inline)) {
      int from[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) from[kb] = sees[kb] - kStage * st - kRows * n - 4 * half;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(
            &lds.shift[wave][kRows * n + 8 * i + 4 * half]);
        const float nl[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const float p = fast_exp2(fmaf(sc[kb][4 * i + j], a.scale_log2, nl[j]));
            acc[kb] += (kMask == 0 || 8 * i + j >= from[kb]) &&
                       (kMask != 2 || nl[j] != -INFINITY) ? p : 0.f;
          }
      }
    };

    // The first stage with a row that sees one of the wave's keys.
    int first = 0;
    if (c.causal)
      first = max(max(key0 - ahead - tok0, 0) * a.group - first_block * kRows, 0) / kStage;
    first = key0 < kv_len ? min(first, stages) : stages;
    for (int st = 0; st < stages; ++st) {
      if (turn == 0) __builtin_amdgcn_s_setprio(0);
      else if (turn == 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(2);
      turn = turn == 2 ? 0 : turn + 1;
      auto load = [&](int ks) __attribute__((always_inline)) {
        if (ks <= kDma) stage_load(ks, (st + 1) & 1);
        if (kSteps <= kDma && ks == kSteps - 1) {
#pragma unroll
          for (int i = kSteps; i <= kDma; ++i) stage_load(i, (st + 1) & 1);
        }
      };
      if (st < first) {
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) load(ks);
      } else {
        const float lse = lds.lse[st & 1][wave][lane];
        scores(0, load);
        // (Rows behind the last one are copies of its token's that give nothing.)
        int tok, head;
        split(my_first + lane, tok, head);
        const bool there = my_base + tok <= last_tok && lse != -INFINITY;
        lds.shift[wave][lane] = there ? lse * -kLog2e : -INFINITY;
        const uint64_t none = __builtin_amdgcn_ballot_w64(lse == -INFINITY);
        auto block_exps = [&](int n) __attribute__((always_inline)) {
          if (uint32_t(none >> (32 * n)) != 0) exps(std::integral_constant<int, 2>{}, st, n);
          else if (partly(n)) exps(std::integral_constant<int, 1>{}, st, n);
          else exps(std::integral_constant<int, 0>{}, st, n);
        };
        block_exps(0);
        if (2 * st + 1 < blocks) {
          scores(1, [](int) {});
          block_exps(1);
        }
      }
      stage_prepare();
      advance();
      q_at ^= kStage * kRow;
      // The next stage is here and this one has been read: the one after it is loaded
      // over it.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const float w = acc[kb] + __shfl_xor(acc[kb], 32);
      const int key = key0 + 32 * kb + r;
      if (half != 0 || key >= kv_len) continue;
      if (z.z >= 0) {
        c.parts[int64_t(z.z) * kUnitKeys + key - key_first] = w;
        continue;
      }
      if (block[kb] >= 0) store_weight(a, block[kb], h, key, y.z, w, key >= y.w);
    }
    u = rfl(z.w);
  } while (u != 0);
}

// Sums of the units whose rows were cut: a workgroup per (key tile, KV head), a
// thread per key, the partials in order.  Record: KV head, first key, partials, kv_len |
// first partial, page offset, request, first new key.
__global__ __launch_bounds__(kUnitKeys) void weights_join_kernel(ChunkArgs c, const int4* joins) {
  const int4 x = joins[2 * blockIdx.x], y = joins[2 * blockIdx.x + 1];
  const int key = x.y + threadIdx.x;
  if (key >= x.w) return;
  const float* p = c.parts + int64_t(y.x) * kUnitKeys + threadIdx.x;
  float w = 0.f;
  int i = 0;
  for (; i + 4 <= x.z; i += 4) {                    // four loads in flight
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = p[int64_t(i + j) * kUnitKeys];
#pragma unroll
    for (int j = 0; j < 4; ++j) w += v[j];
  }
  for (; i < x.z; ++i) w += p[int64_t(i) * kUnitKeys];
  const int32_t block = block_of(c.w, int64_t(y.y) + key / kPage);
  if (block >= 0) store_weight(c.w, block, x.x, key, y.z, w, key >= y.w);
}

struct TokenArgs {
  WeightsArgs w;
  const int32_t* indptr;           // [batch + 1] pages
  const int32_t* last_page_len;
  int32_t batch;
};

constexpr int kTokenThreads = 256;
constexpr int64_t kTokenWorkgroups = 512;   // two per CU: what its registers hold
// Pages per task: 64 registers of K, twice; at head_dim 256 32, as its query takes 32 more
// (two pages spilled, and a reload waits for all of K: 64 requests of 512 to 4096
// tokens 141 us, 129 to 132 with one).
constexpr int token_pages(int head_dim) { return head_dim == 256 ? 1 : 512 / head_dim; }

// A wave runs every so-manieth task; a task is kPages consecutive entries of the
// batch's page list for one KV head (heads fastest: neighbouring waves read the same
// tokens' rows at the same time).  Bound by memory: a task's K (16 KB), old scores and
// query are loaded while the one before is computed, its page ids a task earlier
// still.  S = Q K^T per page with v_mfma_f32_16x16x32 (A: lane l = row l%16, k =
// 8(l/16)..+7; B: column l%16; C: acc[j] = row 4(l/16)+j, column l%16): rows are the
// group's query heads, columns the page's tokens.  Lane 16 i + r then owns token r of
// page i.  64 requests of 512 to 4096 tokens, 32 / 8 heads of 128: 288 MB in 58 us, 5.0
// TB/s (the decode kernels' non-temporal loads of whole pages reach 6.2 to 7.0).
template <typename T, int D>
__global__ __launch_bounds__(kTokenThreads, 2) void weights_token_kernel(TokenArgs c) {
  constexpr int kSteps = D / 32;
  constexpr int kPages = token_pages(D);
  constexpr int kSets = (kPages + 3) / 4;     // of four pages, a quarter wave each
  typedef typename T::x8 x8;
  const WeightsArgs& a = c.w;
  const int lane = threadIdx.x & 63, r = lane & 15, quad = lane >> 4;
  const int Hq = a.num_kv_heads * a.group;
  const int64_t pages = min(int64_t(c.indptr[c.batch]), a.num_indices);
  const int64_t tasks = (pages + kPages - 1) / kPages * a.num_kv_heads;
  const int64_t waves = int64_t(gridDim.x) * (kTokenThreads / 64);
  const int64_t wave = int64_t(blockIdx.x) * (kTokenThreads / 64) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t t = wave;
  if (t >= tasks) return;
  // The first 64 requests' pages and last pages' tokens, a lane each (a load of them
  // beside a task would wait for the next one's K); further requests' are read.
  const int begin0 = lane < c.batch ? c.indptr[lane] : INT32_MAX;
  const int end0 = lane < c.batch ? c.indptr[lane + 1] : INT32_MAX;
  const int lpl0 = lane < c.batch ? c.last_page_len[lane] : 0;
  struct Request { int first, end, lpl; };
  auto request = [&](int b) __attribute__((always_inline)) {
    if (b < 64)
      return Request{__builtin_amdgcn_readlane(begin0, b), __builtin_amdgcn_readlane(end0, b),
                     __builtin_amdgcn_readlane(lpl0, b)};
    return Request{c.indptr[b], c.indptr[b + 1], c.last_page_len[b]};
  };

  struct Task { int h; int64_t p0; };
  auto task_of = [&](int64_t i) __attribute__((always_inline)) {
    const int64_t g = i / a.num_kv_heads;
    return Task{int(i - g * a.num_kv_heads), g * kPages};
  };
  // Lane i < kPages: page i's id as in the list (the last one's past its end).
  auto load_ids = [&](const Task& k) __attribute__((always_inline)) {
    return a.indices[min(k.p0 + lane % kPages, pages - 1)];
  };
  // The request of a page: the first whose pages end behind it (uniform).
  auto request_of = [&](int64_t p) __attribute__((always_inline)) {
    int b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end0 <= p));
    for (int base = 64; b == base && base < c.batch; base += 64) {
      const int at = base + lane;
      b += __builtin_popcountll(
          __builtin_amdgcn_ballot_w64(at < c.batch && c.indptr[at + 1] <= p));
    }
    return b;
  };
  struct Loaded {
    x8 k[kPages][kSteps];
    x8 q[kSteps];          // the first 16 query heads of the first page's request
    float lse[4];          // and the lane's four rows' lse
    float old[kSets];      // the lane's tokens' scores
    int32_t block[kSets];  // the lane's pages' blocks, -1: missing or past the list
    int b;                 // request of the first page
  };
  auto load_q = [&](int b, int h, int g0, x8 (&q)[kSteps], float (&lse)[4])
      __attribute__((always_inline)) {
    const int n = min(16, a.group - g0);
    const uint16_t* qp = a.q + int64_t(b) * a.q_stride +
                         (int64_t(h) * a.group + g0 + min(r, n - 1)) * D + 8 * quad;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks)
      q[ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(qp + 32 * ks));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      lse[j] = a.lse[int64_t(b) * Hq + h * a.group + g0 + min(4 * quad + j, n - 1)];
  };
  auto load = [&](const Task& k, int32_t ids, Loaded& x) __attribute__((always_inline)) {
    const int32_t id = uint64_t(ids) < uint64_t(a.num_blocks) ? ids : -1;
#pragma unroll
    for (int i = 0; i < kPages; ++i) {
      const int32_t blk = max(__builtin_amdgcn_readlane(id, i), 0);   // (block 0 if missing)
      const uint16_t* kp = a.k_cache + int64_t(blk) * a.block_stride + k.h * D +
                           r * a.token_stride + 8 * quad;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
        x.k[i][ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(kp + 32 * ks));
    }
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      const int page = 4 * i + quad;
      const int32_t blk = __shfl(id, page);
      x.block[i] = page < kPages && k.p0 + page < pages ? blk : -1;
      x.old[i] = a.scores[(int64_t(max(x.block[i], 0)) * a.num_kv_heads + k.h) * kPage + r];
    }
    x.b = min(request_of(k.p0), c.batch - 1);
    load_q(x.b, k.h, 0, x.q, x.lse);
  };

  // (Ids come before the K loads that were issued last: waiting for them does not
  // wait for those.)
  Task now = task_of(t), next = task_of(min(t + waves, tasks - 1));
  int32_t ids0 = load_ids(now), ids = load_ids(next);
  Loaded x;
  load(now, ids0, x);
  for (; t < tasks; t += waves) {
    Loaded y;
    const Task after = task_of(min(t + 2 * waves, tasks - 1));
    const int32_t ids2 = load_ids(after);
    if (t + waves < tasks) load(next, ids, y);
    ids = ids2;
    int b = x.b;
    Request req = request(b);
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      float mine = 0.f;
      bool fresh = false, in = false;
      int key = 0, owner = 0;
#pragma unroll
      for (int i = 4 * set; i < min(kPages, 4 * set + 4); ++i) {
        const int64_t p = now.p0 + i;
        if (p >= pages) continue;
        if (p >= req.end) {       // this page is another request's
          b = request_of(p);
          if (b >= c.batch) break;
          req = request(b);
          load_q(b, now.h, 0, x.q, x.lse);
        }
        const int first = req.first, last = req.end - 1;
        // (a page in front of the first request's has none)
        const int tokens = p < first ? 0 : p < last ? kPage : req.lpl;
        float w = 0.f;
        for (int g0 = 0; g0 < a.group; g0 += 16) {
          if (g0 > 0) load_q(b, now.h, g0, x.q, x.lse);
          f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks) s = T::mfma16(x.q[ks], x.k[i][ks], s);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = fast_exp2(fmaf(s[j], a.scale_log2, x.lse[j] * -kLog2e));
            w += 4 * quad + j < a.group - g0 && x.lse[j] != -INFINITY ? e : 0.f;
          }
        }
        if (a.group > 16) load_q(b, now.h, 0, x.q, x.lse);   // for the next page
        w += __shfl_xor(w, 16);
        w += __shfl_xor(w, 32);
        if (quad == i - 4 * set) {
          mine = w;
          in = r < tokens;
          fresh = p == last && r == tokens - 1;
          key = int(p - first) * kPage + r;
          owner = b;
        }
      }
      if (in && x.block[set] >= 0) {
        const int64_t at = (int64_t(x.block[set]) * a.num_kv_heads + now.h) * kPage + r;
        a.scores[at] = fresh ? mine : x.old[set] + mine;
        if (fresh && a.positions) a.positions[at] = key + first_position(a, owner);
      }
    }
    x = y;
    now = next;
    next = after;
  }
}

constexpr int kMaxGroup = 128;
// Workgroups of the chunk kernel that the chip holds at a time (registers).
int resident(int head_dim) { return head_dim == 64 ? 1024 : head_dim == 128 ? 768 : 512; }
// Costs in row blocks: a unit's start (its K), the join kernel, the least piece of a cut.
constexpr int64_t kUnitCost = 4;
constexpr int64_t kJoinCost = 5;
constexpr int64_t kMinPiece = 4;

// Plan image: units, then joins.
int64_t weights_plan_ints(const kvc_weights_schedule& s) {
  return int64_t(s.num_units) * kRecInts + int64_t(s.num_joins) * kJoinInts;
}

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
  int64_t total_kv = 0;
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
    total_kv += kv_len;
  }
  KVC_REQUIRE((total_kv / kUnitKeys + batch) * hkv < (int64_t(1) << 24), KVC_ERR_INVALID_ARG,
              "too many (key tile, KV head) units");
  // Key tiles: (request, first key, row blocks that see it).
  struct Tile { int b, key0, blocks, new_from; };
  std::vector<Tile> tiles;
  int64_t total = 0;
  for (int b = 0; b < batch; ++b) {
    const int q_len = qo_indptr[b + 1] - qo_indptr[b];
    const int pages = kv_indptr[b + 1] - kv_indptr[b];
    const int kv_len = pages > 0 ? (pages - 1) * kPage + lpl[b] : 0;
    const int fresh = new_tokens ? new_tokens[b] : q_len;
    if (q_len == 0 && fresh == 0) continue;
    // Without queries only the new tokens change (to 0).
    for (int k0 = q_len ? 0 : (kv_len - fresh) / kUnitKeys * kUnitKeys; k0 < kv_len;
         k0 += kUnitKeys) {
      const int64_t n = int64_t(q_len - first_token(k0, q_len, kv_len, causal)) * group;
      const int blocks = q_len ? int((n + kRows - 1) / kRows) : 0;
      tiles.push_back(Tile{b, k0, blocks, kv_len - fresh});
      total += blocks;
    }
  }
  // Either every tile is a unit, or the tiles' blocks are lined up and cut into as
  // many shares of equal cost as workgroups fit, each a few pieces of tiles: what
  // ends sooner.  Whole tiles, longest first, end within the sum of the longest of
  // each round, and within the longest on top of an equal share.
  std::vector<int64_t> by_cost;
  for (const Tile& t : tiles) by_cost.push_back(t.blocks + kUnitCost);
  std::sort(by_cost.begin(), by_cost.end(), std::greater<int64_t>());
  const int64_t wgs_max = resident(head_dim);
  const int64_t cost = (total + int64_t(tiles.size()) * kUnitCost) * hkv;
  int64_t whole = 0;
  for (size_t i = 0; i * wgs_max < tiles.size() * hkv; ++i) whole += by_cost[i * wgs_max / hkv];
  if (!tiles.empty()) whole = std::min(whole, by_cost[0] + (cost - by_cost[0]) / wgs_max);
  const int64_t shares = std::min(wgs_max, total * hkv / kMinPiece);
  const bool cut = shares > 0 && whole > cost / shares + kUnitCost + kMinPiece / 2 + kJoinCost;
  typedef std::array<int32_t, kRecInts> Rec;
  std::vector<Rec> units;
  std::vector<std::array<int32_t, kJoinInts>> joins;
  std::vector<std::array<int32_t, 2>> wgs;       // (first unit, units) by workgroup
  int64_t n_parts = 0;
  auto piece = [&](const Tile& t, int h, int from, int blocks) {
    const int kv_len = (kv_indptr[t.b + 1] - kv_indptr[t.b] - 1) * kPage + lpl[t.b];
    return Rec{h, t.key0, qo_indptr[t.b + 1] - qo_indptr[t.b], kv_len, qo_indptr[t.b],
               kv_indptr[t.b], t.b, t.new_from, from, blocks, -1, 0};
  };
  // Workgroup w runs on XCD w % 8: a request's units of one head, which read the
  // same Q and K, go to one XCD.
  std::vector<Rec> list[8];
  int64_t load[8] = {0};
  int64_t share = 0, used = 0, taken = 0, left_cost = cost;
  std::vector<std::array<int32_t, 2>> by_share(cut ? shares : 0, std::array<int32_t, 2>{0, 0});
  for (size_t t0 = 0; t0 < tiles.size();) {
    size_t t1 = t0;
    while (t1 < tiles.size() && tiles[t1].b == tiles[t0].b) ++t1;
    for (int h = 0; h < hkv; ++h) {
      const int xcd = int(std::min_element(load, load + 8) - load);
      for (size_t i = t0; i < t1; ++i) {
        const Tile& t = tiles[i];
        if (!cut) {
          list[xcd].push_back(piece(t, h, 0, t.blocks));
          load[xcd] += t.blocks + kUnitCost;
          continue;
        }
        const size_t first = units.size();
        int done = 0;
        do {
          const int64_t target = left_cost / (shares - share) + kUnitCost;
          int64_t n = t.blocks - done;
          if (share + 1 < shares) {
            const int64_t want = std::max(kMinPiece, target - used - kUnitCost);
            if (n - want >= kMinPiece) n = want;
          }
          if (by_share[share][1]++ == 0) by_share[share][0] = int32_t(units.size());
          units.push_back(piece(t, h, done, int(n)));
          taken += n + (done == 0 ? kUnitCost : 0);
          used += n + kUnitCost;
          done += int(n);
          if (share + 1 < shares && used + kUnitCost + kMinPiece > target) {
            ++share;
            left_cost -= taken;
            used = taken = 0;
          }
        } while (done < t.blocks);
        const int64_t k = int64_t(units.size() - first);
        if (k == 1) continue;
        joins.push_back({h, t.key0, int32_t(k), units[first][3], int32_t(n_parts),
                         kv_indptr[t.b], t.b, t.new_from});
        for (int64_t j = 0; j < k; ++j) units[first + j][10] = int32_t(n_parts++);
      }
    }
    t0 = t1;
  }
  if (cut) {
    while (!by_share.empty() && by_share.back()[1] == 0) by_share.pop_back();
    const int64_t n = by_share.size();
    for (int64_t w = 0; w < n; ++w) {            // XCD x has the x-th eighth of the shares
      const int64_t x = w % 8;
      wgs.push_back(by_share[x * (n / 8) + std::min(x, n % 8) + w / 8]);
    }
  } else {                                       // longest first in each XCD
    size_t most = 0;
    for (auto& l : list) {
      std::stable_sort(l.begin(), l.end(), [](const Rec& p, const Rec& q) { return p[9] > q[9]; });
      most = std::max(most, l.size());
    }
    for (size_t i = 0; i < most; ++i)
      for (auto& l : list)
        if (i < l.size()) {
          wgs.push_back({int32_t(units.size()), 1});
          units.push_back(l[i]);
        }
  }
  KVC_REQUIRE(units.size() < size_t(1) << 26, KVC_ERR_INVALID_ARG, "too many units");
  sched->batch = batch;
  sched->num_qo_heads = hq;
  sched->num_kv_heads = hkv;
  sched->head_dim = head_dim;
  sched->page_size = page_size;
  sched->causal = causal ? 1 : 0;
  sched->num_units = int32_t(units.size());
  sched->num_parts = int32_t(n_parts);
  sched->num_joins = int32_t(joins.size());
  sched->num_workgroups = int32_t(wgs.size());
  sched->total_q = batch ? qo_indptr[batch] : 0;
  sched->plan_ints = weights_plan_ints(*sched);
  sched->workspace_bytes = n_parts * kUnitKeys * 4;
  KVC_REQUIRE(plan_capacity >= sched->plan_ints && (plan_host || sched->plan_ints == 0),
              KVC_ERR_WORKSPACE,
              "plan buffer too small: need " + std::to_string(sched->plan_ints) + " int32");
  // Every workgroup's first unit, then the others, linked.
  int64_t more = int64_t(wgs.size());
  for (size_t w = 0; w < wgs.size(); ++w) {
    int32_t* at = plan_host + w * kRecInts;
    for (int32_t i = 0; i < wgs[w][1]; ++i) {
      if (i > 0) {
        at[kRecInts - 1] = int32_t(more);
        at = plan_host + more++ * kRecInts;
      }
      std::copy(units[wgs[w][0] + i].begin(), units[wgs[w][0] + i].end(), at);
    }
  }
  int32_t* dst = plan_host + units.size() * kRecInts;
  for (const auto& r : joins) dst = std::copy(r.begin(), r.end(), dst);
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
  KVC_REQUIRE(a.q_stride < (int64_t(1) << 25), KVC_ERR_UNSUPPORTED,
              std::string(who) + ": q token stride of 2^25 elements or more");
  KVC_REQUIRE(!a.offsets || a.num_offsets >= 0, KVC_ERR_INVALID_ARG,
              std::string(who) + ": negative num_offsets");
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
    const kvc_weights_schedule* sched, const int32_t* plan, void* workspace,
    int64_t workspace_bytes, const void* q,
    int64_t q_token_stride, const float* lse, const void* key_cache,
    int64_t cache_block_stride, int64_t cache_token_stride, int64_t num_blocks,
    const int32_t* indices, int64_t num_indices, int32_t dtype, float sm_scale, float* scores,
    int32_t* positions, const int32_t* position_offsets, int32_t num_offsets,
    const int32_t* seq_ids, void* stream) {
  KVC_REQUIRE(sched, KVC_ERR_INVALID_ARG, "null schedule");
  const int Hq = sched->num_qo_heads, Hkv = sched->num_kv_heads, D = sched->head_dim;
  KVC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= kMaxGroup &&
                  (D == 64 || D == 128 || D == 256) && sched->page_size == kPage &&
                  sched->num_units >= 0 && sched->num_parts >= 0 && sched->num_joins >= 0 &&
                  sched->workspace_bytes == int64_t(sched->num_parts) * kUnitKeys * 4 &&
                  sched->num_workgroups >= 0 && sched->num_workgroups <= sched->num_units &&
                  sched->plan_ints == weights_plan_ints(*sched),
              KVC_ERR_INVALID_ARG, "schedule not produced by kvc_weights_plan");
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");
  KVC_REQUIRE(sm_scale > 0.f && std::isfinite(sm_scale), KVC_ERR_INVALID_ARG,
              "sm_scale must be positive and finite");
  if (sched->num_units == 0) return ok();
  KVC_REQUIRE(plan && (sched->total_q == 0 || (q && lse)), KVC_ERR_INVALID_ARG, "null pointer");
  KVC_REQUIRE(aligned(plan, 16), KVC_ERR_ALIGNMENT, "plan must be 16-byte aligned");
  KVC_REQUIRE(sched->num_parts == 0 || (workspace && workspace_bytes >= sched->workspace_bytes),
              KVC_ERR_WORKSPACE,
              "workspace too small: need " + std::to_string(sched->workspace_bytes) + " bytes");
  KVC_REQUIRE(aligned(workspace, 4), KVC_ERR_ALIGNMENT, "workspace must be 4-byte aligned");
  ChunkArgs c;
  c.w = WeightsArgs{static_cast<const uint16_t*>(q), q_token_stride, lse,
                    static_cast<const uint16_t*>(key_cache), cache_block_stride,
                    cache_token_stride, num_blocks, indices, num_indices, Hkv, Hq / Hkv,
                    sm_scale * kLog2e, scores, positions, position_offsets,
                    num_offsets, seq_ids};
  if (const int st = check_common(c.w, Hq, Hkv, D, "kvc_batch_attention_weights_run")) return st;
  c.units = reinterpret_cast<const int4*>(plan);
  c.parts = static_cast<float*>(workspace);
  c.causal = sched->causal;
  const dim3 grid(static_cast<unsigned>(sched->num_workgroups));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto t) {
    typedef decltype(t) T;
    if (D == 64) weights_chunk_kernel<T, 64><<<grid, kChunkThreads, 0, s>>>(c);
    else if (D == 128) weights_chunk_kernel<T, 128><<<grid, kChunkThreads, 0, s>>>(c);
    else weights_chunk_kernel<T, 256><<<grid, kChunkThreads, 0, s>>>(c);
  };
  if (dtype == KVC_DTYPE_BF16) launch(Bf16{});
  else launch(Fp16{});
  KVC_LAUNCH_CHECK();
  if (sched->num_joins > 0) {
    weights_join_kernel<<<dim3(unsigned(sched->num_joins)), kUnitKeys, 0, s>>>(
        c, reinterpret_cast<const int4*>(plan + int64_t(sched->num_units) * kRecInts));
    KVC_LAUNCH_CHECK();
  }
  return ok();
}

extern "C" int kvc_decode_attention_weights(
    const void* q, int64_t q_token_stride, const float* lse, const void* key_cache,
    int64_t cache_block_stride, int64_t cache_token_stride, int64_t num_blocks,
    const int32_t* indptr, const int32_t* indices, int64_t num_indices,
    const int32_t* last_page_len, int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t page_size, int32_t dtype, float sm_scale, float* scores,
    int32_t* positions, const int32_t* position_offsets, int32_t num_offsets,
    const int32_t* seq_ids, void* stream) {
  const int Hq = num_qo_heads, Hkv = num_kv_heads, D = head_dim;
  KVC_REQUIRE(batch >= 0, KVC_ERR_INVALID_ARG, "negative batch");
  KVC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, KVC_ERR_INVALID_ARG,
              "num_qo_heads must be a positive multiple of num_kv_heads");
  KVC_REQUIRE((D == 64 || D == 128 || D == 256) && page_size == kPage && Hq / Hkv <= kMaxGroup,
              KVC_ERR_UNSUPPORTED, "attention weights support head_dim 64, 128, 256, page_size "
                                   "16 and groups up to 128");
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");
  KVC_REQUIRE(sm_scale > 0.f && std::isfinite(sm_scale), KVC_ERR_INVALID_ARG,
              "sm_scale must be positive and finite");
  if (batch == 0 || num_indices == 0) return ok();
  KVC_REQUIRE(q && lse && indptr && last_page_len, KVC_ERR_INVALID_ARG, "null pointer");
  TokenArgs c;
  c.w = WeightsArgs{static_cast<const uint16_t*>(q), q_token_stride, lse,
                    static_cast<const uint16_t*>(key_cache), cache_block_stride,
                    cache_token_stride, num_blocks, indices, num_indices, Hkv, Hq / Hkv,
                    sm_scale * kLog2e, scores, positions, position_offsets,
                    num_offsets, seq_ids};
  if (const int st = check_common(c.w, Hq, Hkv, D, "kvc_decode_attention_weights")) return st;
  c.indptr = indptr;
  c.last_page_len = last_page_len;
  c.batch = batch;
  const int64_t tasks = (num_indices + token_pages(D) - 1) / token_pages(D) * Hkv;
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
