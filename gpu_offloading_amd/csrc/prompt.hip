// Attention of whole prompts over their own contiguous K/V (MFMA, gfx950):
// sequences packed one after another, causal or full, grouped heads.
//
//   s_ij = scale q_i . k_j   (j <= i + kv_len - q_len where causal)
//   out_i = sum_j e^(s_ij - m_i) v_j / l_i,   l_i = sum_j e^(s_ij - m_i),   lse_i = m_i + ln l_i
// in one pass over the keys with a running maximum m and sum l (online softmax), both
// fp32.  The exponentials are rounded to the element type for the second product, as
// the matrix instructions take them in that type: half a step each, independent from
// key to key, which moves an output by about as much as its own rounding does.  l and
// lse are sums of the unrounded ones.
//
// Work unit = (sequence, tile of query rows) x one KV head.  A query row is a
// (token, query head) pair: the `group` query heads of a KV head are packed into
// the rows of a tile, so that each K/V tile staged in LDS serves all of them and
// the causal edge is as narrow as the tile has tokens.  Any group: row r is token
// r / group, head r % group.
#include "kvc_common.h"

#include <algorithm>
#include <array>
#include <cmath>
#include <functional>
#include <type_traits>
#include <utility>
#include <vector>

namespace kvc {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int kWaveRows = 32;                 // query rows per wave
// Keys per tile: at head_dim 64 a tile of 128, whose phases are as long as those of
// 64 keys at head_dim 128 (with 64 keys the barriers and the phases' starts are a
// quarter of them).
constexpr int tile_keys(int head_dim) { return head_dim == 64 ? 128 : 64; }
constexpr int kMaxGroup = 128;
// Waves of a workgroup: two per SIMD, or one with the whole register file
// (head_dim 256: O alone is 128 registers).
constexpr int kWaves(int head_dim) { return head_dim == 256 ? 4 : 8; }
constexpr int tile_rows(int head_dim) { return kWaves(head_dim) * kWaveRows; }
// Word 3 of a raw buffer resource (32-bit data, no swizzle): loads past
// num_records return zeros.
constexpr int kBufferRsrcWord3 = 0x00020000;
// s_waitcnt vmcnt(0) with the other counters unconstrained (gfx9 encoding).
constexpr int kWaitVmcnt0 = 0x0F70;
constexpr float kRescaleLog2 = 8.f;           // lazy-rescale threshold (base 2)
constexpr float kLargeLog2 = 16777216.f;      // 2^24: a maximum's rounding passes 1/2
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, k_stride, v_stride;   // elements between tokens
  const int2* wg_units;                   // [workgroups]: (first unit, units)
  const int4* units;                      // [units][2]: (KV head, first query, q_len, kv_len),
                                          //             (q offset, k offset, key tiles, part)
  int32_t num_kv_heads, group, tile_tokens, causal;
  uint32_t inv_group;                     // 65536 / group, rounded up
  float scale_log2;                       // sm_scale * log2(e)
  uint16_t* out;
  int64_t out_stride;
  float* lse;                             // [total_q][Hq] natural log, may be null
  float* parts;                           // [parts][tile rows][D] outputs of units' pieces
  float* part_max;                        // [parts][tile rows] the maximum m under their sums
};

// The element types: bf16 and fp16 through the same kernel.
struct Bf16 {
  typedef __bf16 e;
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExp = 0x7f80u;   // exponent bits: all set is inf or NaN
  static __device__ __forceinline__ f32x16_t mfma(x8 a, x8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
struct Fp16 {
  typedef _Float16 e;
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExp = 0x7c00u;
  static __device__ __forceinline__ f32x16_t mfma(x8 a, x8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Two floats as a pair of the element type, round to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const typename T::x2 v = {static_cast<typename T::e>(lo), static_cast<typename T::e>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}

// A word with its elements that are inf or NaN made 0; *found is set if there was one.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w, bool* found) {
  const bool lo = (w & T::kExp) == T::kExp, hi = ((w >> 16) & T::kExp) == T::kExp;
  *found |= lo | hi;
  return (lo ? 0u : w & 0xffffu) | (hi ? 0u : w & 0xffff0000u);
}

// LDS tiles hold [key][dim] rows whose 16-byte chunks are XOR-swizzled by key,
// so that MFMA operand reads hit distinct banks: K is read as 16 bytes of one
// key's dims, 16 consecutive keys at a time; V^T through the transposing
// ds_read_b64_tr_b16, 64 bytes of four consecutive keys at a time.  Rows of 128
// bytes (D = 64) put two keys into the 256 bytes of all banks.
template <int D>
__device__ __forceinline__ int k_slot(int key, int chunk) {
  return D == 64 ? chunk ^ ((key >> 1) & 7) : chunk ^ (key & 15);
}
template <int D>
__device__ __forceinline__ int v_slot(int key, int chunk) {
  return D == 64 ? chunk ^ (4 * ((key >> 1) & 1)) : chunk ^ (4 * (key & 3));
}

// A work unit's record: a tile of query rows of one KV head, against all key tiles that
// they see (part 0) or against a run of them (part p: the piece's place among the
// partials + 1; its keys' offset and length are the run's first key's).
struct Unit { int h, tok0, q_len, kv_len, q_off, k_off, ntiles, part; };

// The maximum to subtract from a tile's scaled scores, rounded as m = RN(max s * scale)
// is.  fmaf(s, scale, -m) has the exact product in it: the largest score's exponent is
// not 0 but m's rounding, half a step, up to 1/2 below kLargeLog2.  It cancels against
// the sum, but from there on it would soon overflow the exponential, or flush it
// to 0.  There (no model's scores) scores are scaled and rounded first, so that equal ones
// have equal exponents, the largest 0; divided by the scale again they take the common
// path with a maximum of 0.
template <int KB>
__device__ __forceinline__ float settle_scores(f32x16_t (&s)[KB], float m, float scale_log2) {
#pragma clang fp contract(off)
  const bool large = fabsf(m) >= kLargeLog2;
  if (__builtin_amdgcn_ballot_w64(large) == 0) return m;
  const float inv = __builtin_amdgcn_rcpf(scale_log2);   // (at least 2^-104 here)
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float scaled = s[b][e] * scale_log2;
      s[b][e] = large ? (scaled - m) * inv : s[b][e];
    }
  return large ? 0.f : m;
}

// Whether the weight of key t (of the unit's) for the lane's row vanishes in the element
// type under the maximum m: lanes l and l^32 each add up half of the dims.
template <typename T, int D>
__device__ __forceinline__ bool weight_vanishes(const PromptArgs& a, const Unit& U, int tok,
                                                int head, int half, int t, float m) {
#pragma clang fp contract(off)
  asm volatile("" : "+v"(tok), "+v"(head), "+v"(half));   // (addresses here, not ahead of all)
  const uint16_t* q = a.q + int64_t(U.q_off + tok) * a.q_stride +
                      int64_t(U.h * a.group + head) * D + half * (D / 2);
  const uint16_t* k = a.k + (int64_t(U.k_off) + t) * a.k_stride + U.h * D + half * (D / 2);
  float dot = 0.f;
#pragma unroll 1
  for (int i = 0; i < D / 2; ++i)
    dot += float(__builtin_bit_cast(typename T::e, q[i])) *
           float(__builtin_bit_cast(typename T::e, k[i]));
  dot += __shfl_xor(dot, 32);
  return float(static_cast<typename T::e>(fast_exp2(dot * a.scale_log2 - m))) == 0.f;
}

// A lane's share of a piece's row (O^T entries as accumulated, normalised), the row's
// maximum m and the sum l under it.  (Their log-sum-exp m + log2 l in one number would
// lose l beside a large m.)  l's 32 bits take the place of the lowest four of dims
// 0 to 7, whose other 20 are far more than the output keeps.
template <int D, int kBlocks>
__device__ __forceinline__ void store_part(const PromptArgs& a, int part, int rows, int row,
                                           int half, const f32x16_t (&o)[kBlocks], float l,
                                           float m) {
  const int64_t at = int64_t(part - 1) * rows + row;
  float* p = a.parts + at * D + 4 * half;
#pragma unroll
  for (int db = 0; db < kBlocks; ++db)
#pragma unroll
    for (int i = db == 0; i < 4; ++i)
      *reinterpret_cast<f32x4_t*>(p + 32 * db + 8 * i) =
          f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
  const uint32_t bits = __float_as_uint(l) >> (16 * half);
  u32x4_t first;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    first[j] = (__float_as_uint(o[0][j]) & ~15u) | (bits >> (4 * j) & 15u);
  *reinterpret_cast<u32x4_t*>(p) = first;
  if (half == 0) a.part_max[at] = m;
}

// l from a piece's dims 0 to 7.
__device__ __forceinline__ float part_sum(u32x4_t lo, u32x4_t hi) {
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) bits |= (lo[j] & 15u) << (4 * j) | (hi[j] & 15u) << (16 + 4 * j);
  return __uint_as_float(bits);
}

// head_dim 64 and 128: eight waves in two teams of four, one workgroup per CU,
// two waves per SIMD: wave w of team 0 and wave w of team 1 share SIMD w.  Each
// team owns 128 query rows and both read the same K/V tiles.  Per tile of keys a
// wave has an MFMA phase M_j (O^T += V_{j-1}^T P_{j-1}^T, then S_j^T = K_j Q^T,
// operands read ahead) and a VALU phase X_j (softmax of S_j into P_j).  Team 1
// runs one phase behind team 0 and every phase (slot) ends on a workgroup barrier,
// so that on each SIMD one wave's matrix instructions run beside the other's
// exponentials:
//   slot 2j: team 0 M_j, team 1 X_{j-1};   slot 2j+1: team 0 X_j, team 1 M_j.
// Team 0 also stages: in slot 2j, between its matrix instructions, each of its waves
// issues the direct-to-LDS loads of its quarter of K_{j+1} and V_j (the buffers were
// last read in slot 2j-1) and waits for them before the barrier that ends slot 2j+1.
// (Issued by the team in its VALU phase they cost 570 cycles of a slot of 1200.)
// A workgroup runs a list of units: while one runs, the next one's record and Q
// are loaded (slot 1), and its first K tile is staged in the slot 2n of this one.
//
// S^T tiles come from v_mfma_f32_32x32x16 (A: lane l = row l%32, k =
// 8(l/32)..+7; B: column l%32, same k; C: acc[4i+j] = row 8i+4(l/32)+j, column
// l%32) with K as A: a lane owns ONE query row (column l%32) and 32 of the tile's
// keys, lane l^32 the other 32.  Its P values are then laid out as the B operand
// of O^T += V^T P^T, keys in the order {4h..4h+3, 8+4h..8+4h+3} for lane half h,
// and O^T's columns are query rows too.
//
// Measured: head_dim 128, bf16, 32 / 8 heads, 4 x 4096 tokens not causal 890 to 932 us
// (1235 to 1179 TFLOP/s from card to card), one causal prompt of 16384 1.84 to 1.89 ms (67% of the
// matrix rate at the 1.7 GHz that the power cap leaves), 64 x 512 203 to 207 us (bound by
// Q and the output at each unit's ends); head_dim 64, fp16, 64 / 8 heads, 8 x 4096 not
// causal 2.29 to 2.37 ms (960 to 927 TFLOP/s; in a slot the vector unit is the bound:
// exponential, maximum, sum and conversion of a score cost 22 cycles beside 16 of
// products; ragged prompts spend nearly half their time around units' ends).
template <typename T, int D>
__global__ __launch_bounds__(512, 1) void prompt_kernel(PromptArgs a) {
  constexpr int kRow = 2 * D;                  // bytes per K or V row
  constexpr int kChunks = kRow / 16;
  constexpr int kSteps = D / 16;               // k-steps of S^T
  constexpr int kBlocks = D / 32;              // 32-dim blocks of O^T
  constexpr int kKeys = tile_keys(D);
  constexpr int KB = kKeys / 32;               // 32-key blocks of S^T
  constexpr int kWaveKeys = kKeys / 4;         // keys that a wave of team 1 stages
  constexpr int kTile = kKeys * kRow;
  constexpr int kORow = kRow + 16;             // bytes per staged output row
  constexpr int kDma = kWaveKeys * kRow / 1024;   // loads per wave and tile
  constexpr int kLaneKeys = 1024 / kRow;       // keys per load
  typedef typename T::x8 x8;
  // One LDS object with the tiles first: operand reads then use immediate
  // offsets.  ostage: each wave's finished rows on their way out, padded so that
  // one instruction's pieces spread over the banks, and before that its next rows of Q on
  // their way in (chunks swizzled as K's).  out_off, q_off: the rows' places in the
  // output and in Q, in bytes from the tile's first (kept in registers, they would
  // spill, and a reload waits for every load and store in flight).  bad: the last unit (by its
  // parity) whose boundary tiles held an inf or NaN in V.
  struct Lds {
    uint8_t k[2][kTile];
    uint8_t v[2][kTile];
    uint8_t ostage[8][kWaveRows * kORow];
    uint32_t out_off[8 * kWaveRows];
    uint32_t q_off[8 * kWaveRows];
    int bad[2];
  };
  __shared__ alignas(16) Lds lds;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = wave >> 2;
  const int sw = wave & 3;                     // team 0: the quarter of a tile it stages
  const int lane = threadIdx.x & 63;
  const int r = lane & 31;
  const int half = lane >> 5;
  const int row = wave * kWaveRows + r;
  const int row_tok = int(row * a.inv_group >> 16);     // row / group
  const int row_head = row - row_tok * a.group;
  const int Hq = a.num_kv_heads * a.group;
  if (threadIdx.x < 2) lds.bad[threadIdx.x] = -1;
  if (half == 0) {
    const bool in_tile = row_tok < a.tile_tokens;
    lds.out_off[row] = in_tile ? uint32_t(row_tok * a.out_stride + row_head * D) * 2 : UINT32_MAX;
    lds.q_off[row] = in_tile ? uint32_t(row_tok * a.q_stride + row_head * D) * 2 : UINT32_MAX;
  }

  const int2 span = a.wg_units[blockIdx.x];
  const int u_first = __builtin_amdgcn_readfirstlane(span.x);
  const int u_count = __builtin_amdgcn_readfirstlane(span.y);
  // A unit's record as loaded (VGPRs, no wait) and as used (SGPRs).
  struct RawUnit { int4 x, y; };
  auto fetch_unit = [&](int u) __attribute__((always_inline)) {
    return RawUnit{a.units[2 * u], a.units[2 * u + 1]};
  };
  auto to_unit = [](const RawUnit& t) __attribute__((always_inline)) {
    auto rfl = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    return Unit{rfl(t.x.x), rfl(t.x.y), rfl(t.x.z), rfl(t.x.w), rfl(t.y.x), rfl(t.y.y),
                rfl(t.y.z), rfl(t.y.w)};
  };
  // Rows of no token read the unit's first one; they are never stored.
  auto load_q = [&](const Unit& U, x8 (&dst)[kSteps]) __attribute__((always_inline)) {
    const bool there = row_tok < a.tile_tokens && U.tok0 + row_tok < U.q_len;
    const uint16_t* qp = a.q + int64_t(U.q_off + U.tok0 + (there ? row_tok : 0)) * a.q_stride +
                         int64_t(U.h * a.group + (there ? row_head : 0)) * D + 8 * half;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks)
      dst[ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(qp + 16 * ks));
  };

  Unit cu = to_unit(fetch_unit(u_first));
  int limit = -1, n_full = 0;
  bool row_ok = false;
  auto set_unit = [&](const Unit& U) __attribute__((always_inline)) {
    cu = U;
    const int tok = U.tok0 + row_tok;
    row_ok = row_tok < a.tile_tokens && tok < U.q_len;
    // Last key this row may see (inclusive); tiles [0, n_full) are seen whole by
    // every row of the unit.
    limit = !row_ok ? -1 : a.causal ? min(tok + U.kv_len - U.q_len, U.kv_len - 1) : U.kv_len - 1;
    const int lim_lo = a.causal ? min(U.tok0 + U.kv_len - U.q_len, U.kv_len - 1) : U.kv_len - 1;
    n_full = max(0, min(U.ntiles, (lim_lo + 1) / kKeys));
  };
  set_unit(cu);
  // (Q is waited for here: where the loads may still be under way by one of its paths, the
  // first score products of every unit wait for all that is, stores included.)
  x8 qb[kSteps];
  load_q(cu, qb);
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);

  // Direct-to-LDS staging: load i of a wave fetches keys kLaneKeys i .. of its quarter,
  // lane L key kLaneKeys i + L / kChunks, the chunk whose swizzled slot is
  // L % kChunks, at these byte offsets from the wave's first key.
  const uint32_t k_bytes = uint32_t(a.k_stride * 2), v_bytes = uint32_t(a.v_stride * 2);
  uint32_t lane_k[kDma], lane_v[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int key = kLaneKeys * i + lane / kChunks;
    lane_k[i] = key * k_bytes + k_slot<D>(key, lane % kChunks) * 16;
    lane_v[i] = key * v_bytes + v_slot<D>(key, lane % kChunks) * 16;
  }
  auto wait_dma = []() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    asm volatile("" ::: "memory");
  };
  auto lds_addr = [](const void* p) __attribute__((always_inline)) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void_t*)p));
  };
  // buffer_load_dwordx4 ... lds: 16 bytes per lane, lane L at LDS offset 16 L
  // from the wave-uniform address in M0; inline assembly, so that the compiler
  // does not make every later LDS read wait for it (each wave waits for its own
  // before the barrier that publishes the tiles).  The resource is bounded to the
  // sequence's last row: rows past it are not read.  No compiler-generated code
  // here uses M0 (tests/test_prompt_m0.py checks the built assembly).
  struct Staging { i32x4_t rsrc; uint32_t to; };
  auto staging = [&](const uint8_t* tile, const uint16_t* base, int64_t stride,
                     uint32_t row_bytes, const Unit& U, int j) __attribute__((always_inline)) {
    const int key0 = j * kKeys + sw * kWaveKeys;
    // (past the unit's last tile nothing is read)
    const int rows = max(0, min(kWaveKeys, min(U.kv_len, U.ntiles * kKeys) - key0));
    const uint64_t p = reinterpret_cast<uint64_t>(base + (int64_t(U.k_off) + key0) * stride +
                                                  U.h * D);
    const int bytes = rows > 0 ? int(uint32_t(rows - 1) * row_bytes + kRow) : 0;
    return Staging{i32x4_t{__builtin_amdgcn_readfirstlane(int(uint32_t(p))),
                           __builtin_amdgcn_readfirstlane(int(uint32_t(p >> 32) & 0xFFFF)),
                           __builtin_amdgcn_readfirstlane(bytes), kBufferRsrcWord3},
                   uint32_t(__builtin_amdgcn_readfirstlane(
                       lds_addr(tile + sw * kWaveKeys * kRow)))};
  };
  auto stage_piece = [](const Staging& g, uint32_t lane_off, int i) __attribute__((always_inline)) {
    if (i == 0)
      asm volatile(KVC_SGPR_WAIT KVC_SET_M0("%0") "buffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "s"(g.to), "v"(lane_off), "s"(g.rsrc) : "memory");
    else
      asm volatile(KVC_SET_M0("%0") "buffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "s"(g.to + 1024 * i), "v"(lane_off), "s"(g.rsrc) : "memory");
  };
  auto staging_k = [&](const Unit& U, int j) __attribute__((always_inline)) {
    return staging(lds.k[j & 1], a.k, a.k_stride, k_bytes, U, j);
  };
  auto staging_v = [&](const Unit& U, int j) __attribute__((always_inline)) {
    return staging(lds.v[j & 1], a.v, a.v_stride, v_bytes, U, j);
  };
  auto dma_k = [&](const Unit& U, int j) __attribute__((always_inline)) {
    const Staging g = staging_k(U, j);
#pragma unroll
    for (int i = 0; i < kDma; ++i) stage_piece(g, lane_k[i], i);
  };
  // A boundary tile's V in LDS (this wave's keys, just staged): inf and NaN
  // and rows past the sequence become 0, as 0 times them must not reach the rows
  // that do not see them; finish_unit gives them to those that do.
  auto clean_v = [&](int j, int stamp) __attribute__((always_inline)) {
    uint8_t* mine = lds.v[j & 1] + sw * kWaveKeys * kRow + 16 * lane;
    // The largest exponent of each half word.
    u16x2_t top = {0, 0};
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(mine + 1024 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = __builtin_elementwise_max(
            top, __builtin_bit_cast(u16x2_t, x[e] & (T::kExp << 16 | T::kExp)));
    }
    const int left = cu.kv_len - (j * kKeys + sw * kWaveKeys);   // keys of the sequence
    if (__builtin_amdgcn_ballot_w64(top[0] == T::kExp || top[1] == T::kExp) != 0 ||
        left < kWaveKeys) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kDma; ++i) {
        uint4* at = reinterpret_cast<uint4*>(mine + 1024 * i);
        uint4 x = *at;
        if (kLaneKeys * i + lane / kChunks >= left) {
          x = make_uint4(0, 0, 0, 0);
        } else {
          x.x = finite2<T>(x.x, &bad);
          x.y = finite2<T>(x.y, &bad);
          x.z = finite2<T>(x.z, &bad);
          x.w = finite2<T>(x.w, &bad);
        }
        *at = x;
      }
      if (bad) lds.bad[stamp & 1] = stamp;
    }
  };

  uint32_t v_rd[kBlocks];
  {
    const int e = (lane >> 2) & 3, q = lane & 3, gp = (lane >> 4) & 1;
#pragma unroll
    for (int db = 0; db < kBlocks; ++db)
      v_rd[db] = (4 * half + e) * kRow +
                 (v_slot<D>(4 * half + e, 4 * db + 2 * gp + (q >> 1)) << 4) + ((q & 1) << 3);
  }
  // Score MFMA i of a tile: k-step i / KB of key block i % KB.  Output MFMA i: key step
  // i / kBlocks, head-dim block i % kBlocks; its V^T operand through two transposing
  // reads (ds_read_b64_tr_b16: within 16 lanes, lane j supplies the address of 4
  // consecutive elements and lane i receives element i%4 of the rows supplied
  // by lanes i/4 + {0,4,8,12}).
  auto k_operand = [&](const uint8_t* buf, int i) __attribute__((always_inline)) {
    return __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(
        buf + (32 * (i % KB) + r) * kRow + (k_slot<D>(r, 2 * (i / KB) + half) << 4)));
  };
  auto v_operand = [&](const uint8_t* buf, int i) __attribute__((always_inline)) {
    const uint8_t* p = buf + v_rd[i % kBlocks] + (i / kBlocks) * 16 * kRow;
    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p));
    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p + 8 * kRow));
    return __builtin_bit_cast(x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x16_t o[kBlocks], s[KB];
#pragma unroll
  for (int db = 0; db < kBlocks; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) s[b][e] = 0.f;
  uint32_t pw[KB][8];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) pw[b][e] = 0u;
  // m_run: the row's running maximum (base 2, scaled); l_half: the running sum of
  // p over this lane's half of the keys (fp32, before p is rounded).
  float m_run = -INFINITY, l_half = 0.f;

  auto mfma_phase = [&](int j, auto do_o_c, auto do_s_c, auto between)
      __attribute__((always_inline)) {
    // One run of MFMAs, each operand read kAhead before its own: the first K operands
    // come in while the last output MFMAs run.
    constexpr int NO = decltype(do_o_c)::value ? 2 * KB * kBlocks : 0;
    constexpr int N = NO + (decltype(do_s_c)::value ? KB * kSteps : 0);
    constexpr int kAhead = 3;
    const uint8_t* vb = lds.v[(j - 1) & 1];
    const uint8_t* kb = lds.k[j & 1];
    const f32x16_t zero = {};
    x8 op[N];
    auto operand = [&](int i) __attribute__((always_inline)) {
      return i < NO ? v_operand(vb, i) : k_operand(kb, i - NO);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) op[i] = operand(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + kAhead < N) op[i + kAhead] = operand(i + kAhead);
      if (i < NO) {
        const int st = i / kBlocks;
        const uint32_t* pp = &pw[st >> 1][4 * (st & 1)];
        const x8 pb = __builtin_bit_cast(x8, make_uint4(pp[0], pp[1], pp[2], pp[3]));
        o[i % kBlocks] = T::mfma(op[i], pb, o[i % kBlocks]);
      } else {
        const int m = i - NO;
        s[m % KB] = T::mfma(op[i], qb[m / KB], m < KB ? zero : s[m % KB]);
      }
      between(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // X_j.  Accumulator entry e of key block b holds key 32b + 8(e/4) + 4half + e%4
  // of the tile; on boundary tiles the scores of keys the row does not see become
  // -inf, in place.  The running maximum of a row moves only when it grew by more
  // than kRescaleLog2 (base 2); otherwise it stays, p < 2^8, and O and l need no
  // rescaling.  Each row decides for itself, so a row's result does not depend
  // on which others share its wave.
  auto valu_phase = [&](int j) __attribute__((always_inline)) {
    if (j >= n_full) {
      const int rel = limit - j * kKeys - 4 * half;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[b][e] = 32 * b + 8 * (e >> 2) + (e & 3) <= rel ? s[b][e] : -INFINITY;
    }
    // Four chains: a dependent instruction waits for the one before.
    float m4[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      m4[c] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * KB; ++i) {
        const int e = 4 * KB * c + i;
        m4[c] = fmaxf(m4[c], s[e >> 4][e & 15]);
      }
    }
    float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    const auto sw2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                      false, false);
    mx = fmaxf(__uint_as_float(sw2[0]), __uint_as_float(sw2[1]));
    const float cand = fmaxf(m_run, mx * a.scale_log2);
    const bool grow = cand > m_run + kRescaleLog2;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float alpha = grow ? fast_exp2(m_run - cand) : 1.f;
      m_run = grow ? cand : m_run;
      l_half *= alpha;
#pragma unroll
      for (int db = 0; db < kBlocks; ++db) o[db] *= alpha;
    }
    const float m_use =                            // no key seen yet: all p are 0
        settle_scores(s, m_run == -INFINITY ? 0.f : m_run, a.scale_log2);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8 * KB; ++i) {
      const int b = i >> 3, e = 2 * (i & 7);
      const float p0 = fast_exp2(fmaf(s[b][e], a.scale_log2, -m_use));
      const float p1 = fast_exp2(fmaf(s[b][e + 1], a.scale_log2, -m_use));
      sum[2 * (i & 1)] += p0;
      sum[2 * (i & 1) + 1] += p1;
      pw[b][e >> 1] = pack2<T>(p0, p1);
      if ((i & 3) == 3) {
        // (the sums here, not behind all exponentials, which would keep every p)
        asm volatile("" : "+v"(sum[0]), "+v"(sum[1]), "+v"(sum[2]), "+v"(sum[3]));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    l_half += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };

  // Q of the next unit, straight into the wave's LDS staging (it is free from one unit's
  // end to the next one's) and read from there where the current one is done with.
  // Loads into the registers, 32 rows' lines each, held up both teams' last slots of a
  // unit, and the waits for them its stores (64 x 512 tokens 211 us with them, 203
  // so).  Rows of no token read the unit's first one.
  constexpr int kQRows = 64 / kChunks;           // rows per load
  struct QRows { const uint8_t* from; uint32_t end, to; };
  auto q_rows = [&](const Unit& U) __attribute__((always_inline)) {
    return QRows{reinterpret_cast<const uint8_t*>(a.q + int64_t(U.q_off + U.tok0) * a.q_stride +
                                                  int64_t(U.h * a.group) * D),
                 uint32_t(min(a.tile_tokens, U.q_len - U.tok0) * a.q_stride) * 2,
                 uint32_t(__builtin_amdgcn_readfirstlane(lds_addr(lds.ostage[wave])))};
  };
  auto q_piece = [&](const QRows& w, int i) __attribute__((always_inline)) {
    const int rr = i * kQRows + lane / kChunks;
    const uint32_t off = lds.q_off[wave * kWaveRows + rr];
    const uint32_t at = (off < w.end ? off : 0) + k_slot<D>(rr, lane % kChunks) * 16;
    if (i == 0)
      asm volatile(KVC_SGPR_WAIT KVC_SET_M0("%0") "global_load_lds_dwordx4 %1, %2"
                   :: "s"(w.to), "v"(at), "s"(w.from) : "memory");
    else
      asm volatile(KVC_SET_M0("%0") "global_load_lds_dwordx4 %1, %2"
                   :: "s"(w.to + 1024 * i), "v"(at), "s"(w.from) : "memory");
  };
  auto read_q = [&]() __attribute__((always_inline)) {
    wait_dma();
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks)
      qb[ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(
          lds.ostage[wave] + r * kRow + k_slot<D>(r, 2 * ks + half) * 16));
  };

  // The unit's rows leave through the wave's LDS staging: a lane holds 8-byte
  // pieces of one row; read back, kChunks lanes hold a whole row.  Non-temporal
  // stores: the output is not read again here, and the caches keep K and V.
  auto finish_unit = [&](int k, auto before_stores) __attribute__((always_inline)) {
    const float l = l_half + __shfl_xor(l_half, 32);
    const float inv = l == 0.f ? 0.f : 1.f / l;    // a row that sees no key: 0
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) o[db] *= inv;
    if (cu.ntiles > 0 && lds.bad[k & 1] == k) {
      // p times an inf or NaN that the row sees: NaN where p vanishes, as a product gives.
      for (int t = n_full * kKeys; t < min(cu.ntiles * kKeys, cu.kv_len); ++t) {
        const uint16_t* vr = a.v + (int64_t(cu.k_off) + t) * a.v_stride + cu.h * D + 4 * half;
        const bool gone = weight_vanishes<T, D>(a, cu, cu.tok0 + (row_ok ? row_tok : 0),
                                                row_ok ? row_head : 0, half, t, m_run);
#pragma unroll
        for (int db = 0; db < kBlocks; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint16_t w = vr[32 * db + 8 * (e >> 2) + (e & 3)];
            if (t <= limit && (w & T::kExp) == T::kExp)
              o[db][e] += gone ? NAN : float(__builtin_bit_cast(typename T::e, w));
          }
      }
    }
    if (cu.part) {
      before_stores();
      store_part<D, kBlocks>(a, cu.part, 8 * kWaveRows, row, half, o, l, m_run);
    } else {
      uint8_t* stg = lds.ostage[wave];
      // O^T entry (db, 4i+j) is head dim 32db + 8i + 4half + j: (db, i) is the row's
      // 16-byte chunk 4db + i and half its 8-byte half.
      uint8_t* wr = stg + r * kORow + 8 * half;
#pragma unroll
      for (int db = 0; db < kBlocks; ++db) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint2*>(wr + 16 * (4 * db + i)) =
              make_uint2(pack2<T>(o[db][4 * i], o[db][4 * i + 1]),
                         pack2<T>(o[db][4 * i + 2], o[db][4 * i + 3]));
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      constexpr int kStoreRows = 64 / kChunks;      // rows per store
      const int c = lane % kChunks;
      uint8_t* obase = reinterpret_cast<uint8_t*>(
          a.out + int64_t(cu.q_off + cu.tok0) * a.out_stride + int64_t(cu.h * a.group) * D);
      before_stores();
      // (a row's place is below that of the first token that is not there)
      const uint32_t end = uint32_t(min(a.tile_tokens, cu.q_len - cu.tok0) * a.out_stride) * 2;
#pragma unroll
      for (int t0 = 0; t0 < kWaveRows / kStoreRows; t0 += 4) {
        uint4 v[4];
        uint32_t off[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = (t0 + i) * kStoreRows + lane / kChunks;
          v[i] = *reinterpret_cast<const uint4*>(stg + rr * kORow + 16 * c);
          off[i] = lds.out_off[wave * kWaveRows + rr];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (off[i] < end) store_stream(obase + (off[i] + uint32_t(16 * c)), v[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (row_ok && a.lse && half == 0)
        a.lse[int64_t(cu.q_off + cu.tok0 + row_tok) * Hq + cu.h * a.group + row_head] =
            l == 0.f ? -INFINITY : (m_run + fast_log2(l)) * kLn2;
    }
#pragma unroll
    for (int db = 0; db < kBlocks; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
    m_run = -INFINITY;
    l_half = 0.f;
  };

  // Each team has its own copy of the unit loop (the team is a compile-time
  // constant), first and last tiles peeled; they only meet the same barriers.  A
  // unit whose first K tile was not staged during the one before (the
  // workgroup's first, or one after a unit without keys) starts with a staging
  // step of its own.
  using yes = std::true_type;
  using no = std::false_type;
  auto run = [&](auto team_c) __attribute__((always_inline)) {
    constexpr int kTeam = decltype(team_c)::value;
    auto mfma = [&](int j, auto do_o_c, auto do_s_c, auto between) __attribute__((always_inline)) {
      __builtin_amdgcn_s_setprio(1);
      mfma_phase(j, do_o_c, do_s_c, between);
      __builtin_amdgcn_s_setprio(0);
    };
    auto nothing = [](int) {};
    // Between the first MFMAs of team 0's M_j: K_{j+1} and V_j on their way.
    Staging gk{}, gv{};
    auto stage_tile = [&](int j) __attribute__((always_inline)) {
      return [&, j](int i) __attribute__((always_inline)) {
        if (i == 0) gk = staging_k(cu, j + 1);
        if (i >= 1 && i <= kDma) stage_piece(gk, lane_k[i - 1], i - 1);
        if (i == kDma + 1) gv = staging_v(cu, j);
        if (i > kDma + 1 && i <= 2 * kDma + 1) stage_piece(gv, lane_v[i - kDma - 2], i - kDma - 2);
      };
    };
    static_assert(KB * kSteps > 2 * kDma + 1, "the loads fit between the MFMAs");
    // Team 0, slot 2j+1 (the loads of Q that slot 1 issues may still run).
    auto staged_all = [&](int j, int k, auto with_q) __attribute__((always_inline)) {
      if (with_q) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kWaveRows / kQRows) : "memory");
      else wait_dma();
      if (j >= n_full) clean_v(j, k);
    };
    Unit nu = u_count > 1 ? to_unit(fetch_unit(u_first + 1)) : cu;  // the next unit
    // The one after, and taken from its registers before the unit's stores (a wait for
    // its load behind them would wait for them).
    RawUnit nnu = fetch_unit(u_first);
    Unit after = cu;
    bool staged = false;
    for (int k = 0; k < u_count; ++k) {
      const bool has_next = k + 1 < u_count;
      const int n = cu.ntiles;
      if (k + 2 < u_count) nnu = fetch_unit(u_first + k + 2);
      if (n > 0) {
        if (kTeam == 0) {
          if (!staged) {
            dma_k(cu, 0);
            wait_dma();
            __syncthreads();
          }
          mfma(0, no{}, yes{}, stage_tile(0));
          __syncthreads();
          {
            const QRows w = q_rows(nu);
#pragma unroll
            for (int i = 0; i < kWaveRows / kQRows; ++i) q_piece(w, i);
          }
          valu_phase(0);
          staged_all(0, k, yes{});
          __syncthreads();
          for (int j = 1; j < n; ++j) {
            mfma(j, yes{}, yes{}, stage_tile(j));
            __syncthreads();
            valu_phase(j);
            staged_all(j, k, no{});
            __syncthreads();
          }
          // Q is not read again in this unit (without a next one it is the same
          // again).  The next unit's first K tile goes into lds.k[0], last read in
          // slot 2n-1 or earlier.
          read_q();
          after = to_unit(nnu);
          mfma(n, yes{}, no{}, [&](int i) __attribute__((always_inline)) {
            if (i == 0) gk = staging_k(nu, 0);
            if (i >= 1 && i <= kDma) stage_piece(gk, lane_k[i - 1], i - 1);
          });
          __syncthreads();
          finish_unit(k, wait_dma);
          __syncthreads();
        } else {
          if (!staged) __syncthreads();
          __syncthreads();
          const QRows w = q_rows(nu);
          mfma(0, no{}, yes{}, [&](int i) __attribute__((always_inline)) {
            if (i >= 1 && i <= kWaveRows / kQRows) q_piece(w, i - 1);
          });
          __syncthreads();
          for (int j = 1; j < n; ++j) {
            valu_phase(j - 1);
            __syncthreads();
            mfma(j, yes{}, yes{}, nothing);
            __syncthreads();
          }
          valu_phase(n - 1);
          read_q();
          after = to_unit(nnu);
          __syncthreads();
          mfma(n, yes{}, no{}, nothing);
          __syncthreads();
          finish_unit(k, [] {});
        }
      } else {
        load_q(nu, qb);
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        after = to_unit(nnu);
        finish_unit(k, [] {});
      }
      if (has_next) {
        staged = n > 0 && nu.ntiles > 0;
        set_unit(nu);
        if (k + 2 < u_count) nu = after;
      }
    }
  };
  if (team == 0) run(std::integral_constant<int, 0>{});
  else run(std::integral_constant<int, 1>{});
}

// head_dim 256: O alone is 128 registers of a wave, so four waves, one per SIMD
// with the whole register file, and no second wave to fill the matrix pipe's
// gaps: each wave does that itself, a tile ahead.  While it runs the 32 matrix
// instructions of S_{j+1}^T = K_{j+1} Q^T it does the softmax of S_j between them
// (about as many cycles), then the 32 of O^T += V_j^T P_j^T.  One barrier per tile:
// behind it K_{j+1} and V_j are in LDS for all, and the loads of K_{j+2} and
// V_{j+1} start into the buffers read last before it.  Measured: bf16, 16 / 8 heads, 4 x
// 4096 tokens not causal 1141 to 1159 us (964 to 949 TFLOP/s); bound by what one wave
// can issue.
//
// x * alpha of an accumulator register.  In plain code the rare rescaling of O would
// pull all of it into the ordinary registers and back in every tile (256 moves).  At
// least eight matrix instructions separate it from those that write O before and read
// it after, more than the wait states that the assembler cannot see to here.
__device__ __forceinline__ float scale_acc(float x, float alpha) {
  float t;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(x), "=&v"(t) : "v"(alpha));
  return x;
}

template <typename T, int D>
__global__ __launch_bounds__(256, 1) void prompt_wide_kernel(PromptArgs a) {
  constexpr int kRow = 2 * D;                  // bytes per K or V row
  constexpr int kChunks = kRow / 16;
  constexpr int kSteps = D / 16;               // k-steps of S^T
  constexpr int kBlocks = D / 32;              // 32-dim blocks of O^T
  constexpr int kKeys = tile_keys(D);
  constexpr int kTile = kKeys * kRow;
  constexpr int kDma = 16 * kRow / 1024;       // loads per wave, 16 keys each
  constexpr int kLaneKeys = 1024 / kRow;       // keys per load
  typedef typename T::x8 x8;
  struct Lds {
    uint8_t v[2][kTile];                       // (first: within reach of an immediate offset)
    uint8_t k[2][kTile];
    int bad[2];
  };
  __shared__ alignas(16) Lds lds;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 31;
  const int half = lane >> 5;
  const int row = wave * kWaveRows + r;
  const int row_tok = int(row * a.inv_group >> 16);     // row / group
  const int row_head = row - row_tok * a.group;
  const int Hq = a.num_kv_heads * a.group;
  if (threadIdx.x < 2) lds.bad[threadIdx.x] = -1;

  const int2 span = a.wg_units[blockIdx.x];
  const int u_first = __builtin_amdgcn_readfirstlane(span.x);
  const int u_count = __builtin_amdgcn_readfirstlane(span.y);
  auto get_unit = [&](int u) __attribute__((always_inline)) {
    const int4 x = a.units[2 * u], y = a.units[2 * u + 1];
    auto rfl = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    return Unit{rfl(x.x), rfl(x.y), rfl(x.z), rfl(x.w), rfl(y.x), rfl(y.y), rfl(y.z),
                rfl(y.w)};
  };
  x8 qb[kSteps];
  // Rows of no token read the unit's first one; they are never stored.
  auto load_q = [&](const Unit& U) __attribute__((always_inline)) {
    const bool there = row_tok < a.tile_tokens && U.tok0 + row_tok < U.q_len;
    const uint16_t* qp = a.q + int64_t(U.q_off + U.tok0 + (there ? row_tok : 0)) * a.q_stride +
                         int64_t(U.h * a.group + (there ? row_head : 0)) * D + 8 * half;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks)
      qb[ks] = __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(qp + 16 * ks));
  };

  // Direct-to-LDS staging as in prompt_kernel, 16 keys a wave.
  const uint32_t k_bytes = uint32_t(a.k_stride * 2), v_bytes = uint32_t(a.v_stride * 2);
  uint32_t lane_k[kDma], lane_v[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int key = kLaneKeys * i + lane / kChunks;
    lane_k[i] = key * k_bytes + k_slot<D>(key, lane % kChunks) * 16;
    lane_v[i] = key * v_bytes + v_slot<D>(key, lane % kChunks) * 16;
  }
  auto wait_dma = []() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    asm volatile("" ::: "memory");
  };
  auto lds_addr = [](const void* p) __attribute__((always_inline)) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void_t*)p));
  };
  auto dma = [&](uint8_t* tile, const uint16_t* base, int64_t stride, uint32_t row_bytes,
                 const uint32_t (&lane_off)[kDma], const Unit& U, int j)
      __attribute__((always_inline)) {
    const int key0 = j * kKeys + wave * 16;
    const int rows = max(0, min(16, U.kv_len - key0));
    const uint64_t p = reinterpret_cast<uint64_t>(base + (int64_t(U.k_off) + key0) * stride +
                                                  U.h * D);
    const int bytes = rows > 0 ? int(uint32_t(rows - 1) * row_bytes + kRow) : 0;
    const i32x4_t rsrc = {__builtin_amdgcn_readfirstlane(int(uint32_t(p))),
                          __builtin_amdgcn_readfirstlane(int(uint32_t(p >> 32) & 0xFFFF)),
                          __builtin_amdgcn_readfirstlane(bytes), kBufferRsrcWord3};
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(tile + wave * 16 * kRow));
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      if (i == 0)
        asm volatile(KVC_SGPR_WAIT KVC_SET_M0("%0") "buffer_load_dwordx4 %1, %2, 0 offen lds"
                     :: "s"(to), "v"(lane_off[i]), "s"(rsrc) : "memory");
      else
        asm volatile(KVC_SET_M0("%0") "buffer_load_dwordx4 %1, %2, 0 offen lds"
                     :: "s"(to + 1024 * i), "v"(lane_off[i]), "s"(rsrc) : "memory");
    }
  };
  auto dma_k = [&](const Unit& U, int j) __attribute__((always_inline)) {
    dma(lds.k[j & 1], a.k, a.k_stride, k_bytes, lane_k, U, j);
  };
  auto dma_v = [&](const Unit& U, int j) __attribute__((always_inline)) {
    dma(lds.v[j & 1], a.v, a.v_stride, v_bytes, lane_v, U, j);
  };
  auto clean_v = [&](const Unit& U, int j, int stamp) __attribute__((always_inline)) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      const int key = kLaneKeys * i + lane / kChunks;
      uint4* at = reinterpret_cast<uint4*>(lds.v[j & 1] + wave * 16 * kRow + 1024 * i + 16 * lane);
      uint4 x = *at;
      if (j * kKeys + wave * 16 + key >= U.kv_len) {
        x = make_uint4(0, 0, 0, 0);
      } else {
        x.x = finite2<T>(x.x, &bad);
        x.y = finite2<T>(x.y, &bad);
        x.z = finite2<T>(x.z, &bad);
        x.w = finite2<T>(x.w, &bad);
      }
      *at = x;
    }
    if (bad) lds.bad[stamp & 1] = stamp;
  };

  uint32_t v_rd[kBlocks];
  {
    const int e = (lane >> 2) & 3, q = lane & 3, gp = (lane >> 4) & 1;
#pragma unroll
    for (int db = 0; db < kBlocks; ++db)
      v_rd[db] = (4 * half + e) * kRow +
                 (v_slot<D>(4 * half + e, 4 * db + 2 * gp + (q >> 1)) << 4) + ((q & 1) << 3);
  }
  auto k_operand = [&](const uint8_t* buf, int i) __attribute__((always_inline)) {
    return __builtin_bit_cast(x8, *reinterpret_cast<const uint4*>(
        buf + (32 * (i & 1) + r) * kRow + (k_slot<D>(r, 2 * (i >> 1) + half) << 4)));
  };
  auto v_operand = [&](const uint8_t* buf, int i) __attribute__((always_inline)) {
    const uint8_t* p = buf + v_rd[i % kBlocks] + (i / kBlocks) * 16 * kRow;
    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p));
    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p + 8 * kRow));
    return __builtin_bit_cast(x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x16_t o[kBlocks], s[2], sn[2];
  uint32_t pw[2][8];
  const f32x16_t zero = {};
  constexpr int kS = 2 * kSteps;               // MFMAs of S^T
  constexpr int kAhead = 4;                    // operands read ahead
  static_assert(kS >= 24, "the softmax's pieces fit between the score MFMAs");

  Unit cu = get_unit(u_first);
  load_q(cu);
  bool staged = false;
  for (int k = 0; k < u_count; ++k) {
    const int n = cu.ntiles;
    const bool has_next = k + 1 < u_count;
    const Unit nu = has_next ? get_unit(u_first + k + 1) : cu;
    const int tok = cu.tok0 + row_tok;
    const bool row_ok = row_tok < a.tile_tokens && tok < cu.q_len;
    const int limit = !row_ok ? -1
                      : a.causal ? min(tok + cu.kv_len - cu.q_len, cu.kv_len - 1) : cu.kv_len - 1;
    // Tiles [0, n_full) are seen whole by every row of the unit.
    const int lim_lo = a.causal ? min(cu.tok0 + cu.kv_len - cu.q_len, cu.kv_len - 1) : cu.kv_len - 1;
    const int n_full = max(0, min(n, (lim_lo + 1) / kKeys));
    // K_0 of the next unit goes into lds.k[0], which the last tile's S_{n} must not
    // read meanwhile: n odd.
    const bool early = n > 0 && has_next && nu.ntiles > 0 && (n & 1);
    float m_run = -INFINITY, l_half = 0.f;
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) o[db] = zero;

    if (n > 0) {
      if (!staged) {
        __syncthreads();        // (the last unit's reads are done)
        dma_k(cu, 0);
      }
      wait_dma();
      __syncthreads();
      if (1 < n) dma_k(cu, 1);
      dma_v(cu, 0);
      {
        x8 kop[kS];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) kop[i] = k_operand(lds.k[0], i);
#pragma unroll
        for (int i = 0; i < kS; ++i) {
          if (i + kAhead < kS) kop[i + kAhead] = k_operand(lds.k[0], i + kAhead);
          s[i & 1] = T::mfma(kop[i], qb[i >> 1], i < 2 ? zero : s[i & 1]);
        }
      }
      // One tile; S of the next one goes to `sn` (behind the last tile that is a
      // product of whatever the buffer holds, which nothing reads).
      auto tile = [&](int j, f32x16_t (&s)[2], f32x16_t (&sn)[2]) __attribute__((always_inline)) {
        wait_dma();
        if (j >= n_full) clean_v(cu, j, k);
        __syncthreads();
        if (j + 2 < n) dma_k(cu, j + 2);
        if (j + 1 < n) dma_v(cu, j + 1);
        // The next unit's first K tile: no K tile of this one is read again but the
        // one in the other buffer.
        if (j + 1 == n && early) dma_k(nu, 0);

        if (j >= n_full) {
          const int rel = limit - j * kKeys - 4 * half;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              s[b][e] = 32 * b + 8 * (e >> 2) + (e & 3) <= rel ? s[b][e] : -INFINITY;
        }
        const uint8_t* kb = lds.k[(j + 1) & 1];
        float mx = -INFINITY, sum = 0.f;
        x8 kop[kS];
        auto score = [&](int i) __attribute__((always_inline)) {
          if (i + kAhead < kS) kop[i + kAhead] = k_operand(kb, i + kAhead);
          sn[i & 1] = T::mfma(kop[i], qb[i >> 1], i < 2 ? zero : sn[i & 1]);
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) kop[i] = k_operand(kb, i);
        // The maximum between the first MFMAs, the exponentials, two a step, between the
        // others.
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          score(i);
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[i >> 2][4 * (i & 3) + e]);
          __builtin_amdgcn_sched_barrier(0);
        }
        const auto sw2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx),
                                                          __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(sw2[0]), __uint_as_float(sw2[1]));
        const float cand = fmaxf(m_run, mx * a.scale_log2);
        const bool grow = cand > m_run + kRescaleLog2;
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
          const float alpha = grow ? fast_exp2(m_run - cand) : 1.f;
          m_run = grow ? cand : m_run;
          l_half *= alpha;
#pragma unroll
          for (int db = 0; db < kBlocks; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[db][e] = scale_acc(o[db][e], alpha);
        }
        const float m_use =                        // no key seen yet: all p are 0
            settle_scores(s, m_run == -INFINITY ? 0.f : m_run, a.scale_log2);
#pragma unroll
        for (int i = 8; i < kS; ++i) {
          score(i);
          if (i < 24) {
            const int b = (i - 8) >> 3, e = 2 * ((i - 8) & 7);
            const float p0 = fast_exp2(fmaf(s[b][e], a.scale_log2, -m_use));
            const float p1 = fast_exp2(fmaf(s[b][e + 1], a.scale_log2, -m_use));
            sum += p0 + p1;
            pw[b][e >> 1] = pack2<T>(p0, p1);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        l_half += sum;
        constexpr int kN = 4 * kBlocks;
        const uint8_t* vb = lds.v[j & 1];
        x8 vop[kN];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) vop[i] = v_operand(vb, i);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (i + kAhead < kN) vop[i + kAhead] = v_operand(vb, i + kAhead);
          const int st = i / kBlocks;
          const uint32_t* pp = &pw[st >> 1][4 * (st & 1)];
          const x8 pb = __builtin_bit_cast(x8, make_uint4(pp[0], pp[1], pp[2], pp[3]));
          o[i % kBlocks] = T::mfma(vop[i], pb, o[i % kBlocks]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      for (int j = 0; j < n; j += 2) {
        tile(j, s, sn);
        if (j + 1 < n) tile(j + 1, sn, s);
      }
    }
    if (has_next) load_q(nu);

    const float l = l_half + __shfl_xor(l_half, 32);
    const float inv = l == 0.f ? 0.f : 1.f / l;    // a row that sees no key: 0
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) o[db] *= inv;
    if (n > 0 && lds.bad[k & 1] == k) {
      // As in prompt_kernel.
      for (int t = n_full * kKeys; t < min(n * kKeys, cu.kv_len); ++t) {
        const uint16_t* vr = a.v + (int64_t(cu.k_off) + t) * a.v_stride + cu.h * D + 4 * half;
        const bool gone = weight_vanishes<T, D>(a, cu, cu.tok0 + (row_ok ? row_tok : 0),
                                                row_ok ? row_head : 0, half, t, m_run);
#pragma unroll
        for (int db = 0; db < kBlocks; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint16_t w = vr[32 * db + 8 * (e >> 2) + (e & 3)];
            if (t <= limit && (w & T::kExp) == T::kExp)
              o[db][e] += gone ? NAN : float(__builtin_bit_cast(typename T::e, w));
          }
      }
    }
    if (cu.part) {
      store_part<D, kBlocks>(a, cu.part, 4 * kWaveRows, row, half, o, l, m_run);
    } else if (row_ok) {
      // O^T entry (db, 4i+j) is head dim 32db + 8i + 4half + j of this lane's row.
      uint16_t* op = a.out + int64_t(cu.q_off + tok) * a.out_stride +
                     int64_t(cu.h * a.group + row_head) * D + 4 * half;
#pragma unroll
      for (int db = 0; db < kBlocks; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint2*>(op + 32 * db + 8 * i) =
              make_uint2(pack2<T>(o[db][4 * i], o[db][4 * i + 1]),
                         pack2<T>(o[db][4 * i + 2], o[db][4 * i + 3]));
      if (a.lse && half == 0)
        a.lse[int64_t(cu.q_off + tok) * Hq + cu.h * a.group + row_head] =
            l == 0.f ? -INFINITY : (m_run + fast_log2(l)) * kLn2;
    }
    staged = early;
    cu = nu;
  }
}

// Units that were cut along their keys: out = sum_i w_i O_i / sum_i w_i over the pieces,
// w_i = l_i 2^(m_i - max m).  A thread per four dims of a row.  Record: KV head, first
// query, q_len, q offset | first partial, pieces, 0, 0.
template <typename T, int D>
__global__ __launch_bounds__(256)
void prompt_join_kernel(PromptArgs a, const int4* joins, int rows) {
  constexpr int kLanes = D / 4;
  const int4 x = joins[2 * blockIdx.x], y = joins[2 * blockIdx.x + 1];
  const int row = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int row_tok = int(row * a.inv_group >> 16), row_head = row - row_tok * a.group;
  const int tok = x.y + row_tok;
  if (row_tok >= a.tile_tokens || tok >= x.z) return;
  const float* pm = a.part_max + int64_t(y.x) * rows + row;
  const u32x4_t* po =
      reinterpret_cast<const u32x4_t*>(a.parts + (int64_t(y.x) * rows + row) * D);
  const uint32_t keep = c < 2 ? ~15u : ~0u;      // (the first dims' lowest bits are l's)
  float m = -INFINITY;
  for (int i = 0; i < y.y; ++i) m = fmaxf(m, pm[int64_t(i) * rows]);
  const float base = m == -INFINITY ? 0.f : m;   // no piece saw a key: all weights are 0
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < y.y; ++i) {
    const u32x4_t* p = po + int64_t(i) * rows * kLanes;
    const float w = part_sum(p[0], p[1]) * fast_exp2(pm[int64_t(i) * rows] - base);
    const u32x4_t v = p[c];
    sum += w;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = fmaf(w, __uint_as_float(v[j] & keep), o[j]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int head = x.x * a.group + row_head;
  *reinterpret_cast<uint2*>(a.out + int64_t(x.w + tok) * a.out_stride + int64_t(head) * D + 4 * c) =
      make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  if (a.lse && c == 0)
    a.lse[int64_t(x.w + tok) * a.num_kv_heads * a.group + head] =
        sum == 0.f ? -INFINITY : (base + fast_log2(sum)) * kLn2;
}

// Persistent workgroups: one per CU of an MI355X.
constexpr int64_t kMaxWorkgroups = 256;
constexpr int kUnitInts = 8;
constexpr int kJoinInts = 8;
// Costs in key tiles: a unit's start and end, what a piece's fp32 output adds to them, the
// join; and the shortest piece.
constexpr int kUnitCost = 3, kPartCost = 3, kJoinCost = 5, kMinPiece = 4;
constexpr int kXcds = 8;
int64_t plan_workgroups(int64_t units) { return std::min(kMaxWorkgroups, units); }
int64_t table_ints(int64_t workgroups) { return (2 * workgroups + 3) / 4 * 4; }

// Plan image: the work list, then the joins' records.
int64_t prompt_plan_ints(const kvc_prompt_schedule& s) {
  return table_ints(s.num_workgroups) + int64_t(s.num_units) * kUnitInts +
         int64_t(s.num_joins) * kJoinInts;
}
int64_t prompt_workspace_bytes(const kvc_prompt_schedule& s) {
  return s.num_parts * tile_rows(s.head_dim) * (s.head_dim + 1) * 4;
}

// The work list: a table of the workgroups' (first unit, units), then the unit
// records in workgroup order.  `rec`: a record per item (entry 0 the sequence, 6 its
// tiles, 7 a piece's place among the `parts` of one head, + 1), sequence by sequence; a
// unit is an item of one KV head.
//
// Workgroup w runs on XCD w % 8, whose L2 serves the K and V of its units: the units
// are lined up sequence by sequence and head by head, and the line is cut into eight
// parts of equal cost, so that a head's K and V go through one XCD (seven heads at
// most through two).  In each part units are dealt in line order, a head's longest
// first, to the least loaded workgroup; the last quarter of a part longest first over
// all its heads, which evens the ends out.  Where units are cut (few of them) they are
// all dealt longest first to all workgroups.
void write_plan(const std::vector<int32_t>& rec, int64_t n, int hkv, int64_t W, int parts_per_head,
                int32_t* plan_host) {
  struct Line { int32_t item, head, cost; };
  const auto longer = [](const Line& x, const Line& y) { return x.cost > y.cost; };
  std::vector<Line> line, seq;
  line.reserve(size_t(n) * hkv);
  int64_t total = 0;
  for (int64_t i = 0; i < n;) {
    const int32_t b = rec[i * kUnitInts];
    seq.clear();
    for (; i < n && rec[i * kUnitInts] == b; ++i) {
      const int32_t* r = rec.data() + i * kUnitInts;
      seq.push_back(Line{int32_t(i), 0, r[6] + kUnitCost + (r[7] ? kPartCost : 0)});
      total += int64_t(seq.back().cost) * hkv;
    }
    std::stable_sort(seq.begin(), seq.end(), longer);
    for (int h = 0; h < hkv; ++h)
      for (const Line& l : seq) line.push_back(Line{l.item, h, l.cost});
  }
  const int parts = W % kXcds == 0 && !parts_per_head ? kXcds : 1;
  // The least loaded workgroup: a heap of load * 256 + workgroup.
  static_assert(kMaxWorkgroups <= 256, "a workgroup's number has 8 bits");
  std::vector<int64_t> heap;
  std::vector<uint8_t> owner(line.size());
  std::vector<int32_t> count(W, 0);
  size_t u = 0;
  int64_t done = 0;
  for (int x = 0; x < parts; ++x) {
    const int64_t from = done, until = total * (x + 1) / parts;
    size_t end = u;
    // Every workgroup gets a unit, and the last part what is left.
    const size_t each = size_t(W / parts), least = u + each;
    const size_t most = line.size() - size_t(parts - 1 - x) * each;
    while (end < most && (end < least || x == parts - 1 || done + line[end].cost / 2 < until))
      done += line[end++].cost;
    size_t tail = end;
    int64_t rest = parts_per_head ? done : (done - from) / 4;
    while (tail > u && rest > 0) rest -= line[--tail].cost;
    std::stable_sort(line.begin() + tail, line.begin() + end, longer);
    heap.clear();
    for (int64_t b = x; b < W; b += parts) heap.push_back(b);
    for (; u < end; ++u) {
      const int wg = int(heap[0] & 255);
      owner[u] = uint8_t(wg);
      ++count[wg];
      const int64_t key = heap[0] + int64_t(line[u].cost) * 256;
      size_t at = 0;
      for (size_t child; (child = 2 * at + 1) < heap.size(); at = child) {
        if (child + 1 < heap.size() && heap[child + 1] < heap[child]) ++child;
        if (heap[child] >= key) break;
        heap[at] = heap[child];
      }
      heap[at] = key;
    }
  }
  const int64_t table = table_ints(W);
  std::fill_n(plan_host, table, 0);
  for (int64_t b = 0, next = 0; b < W; ++b) {
    plan_host[2 * b] = int32_t(next);
    plan_host[2 * b + 1] = count[b];
    next += count[b];
    count[b] = plan_host[2 * b];                 // and on: the place of its next unit
  }
  for (size_t i = 0; i < line.size(); ++i) {
    int32_t* dst = plan_host + table + int64_t(count[owner[i]]++) * kUnitInts;
    std::copy_n(rec.data() + int64_t(line[i].item) * kUnitInts, kUnitInts, dst);
    dst[0] = line[i].head;
    if (dst[7]) dst[7] += line[i].head * parts_per_head;
  }
}

// Time in tiles of items that are units of hkv heads each, longest first on W workgroups:
// within the sum of the longest of each round, and within the longest on top of an
// equal share.
int64_t estimate(std::vector<int>& costs, int hkv, int64_t W) {
  std::sort(costs.begin(), costs.end(), std::greater<int>());
  int64_t total = 0, rounds = 0;
  for (const int c : costs) total += c;
  total *= hkv;
  for (size_t i = 0; i * W < costs.size() * hkv; ++i) rounds += costs[i * W / hkv];
  return std::min(rounds, costs[0] + (total - costs[0]) / W);
}

// How units are cut along their keys: where fewer units than two rounds of workgroups
// leave many of these idle, the items behind the `whole` longest go in pieces of at
// most `longest` tiles (0: none does).  Measured: 8000 tokens of 4 query heads and one KV
// head (125 units) 156 us whole, 84 cut; 4 sequences of 1000 to 1200 at head_dim 256, not
// causal (284 units, two rounds) 92 and 73.
struct Cut { int64_t whole; int longest; };

Cut choose_cut(const std::vector<int>& tiles, int hkv) {
  const int64_t n = int64_t(tiles.size()), W = kMaxWorkgroups;
  if (n == 0 || n * hkv > 2 * W) return Cut{0, 0};
  std::vector<int> costs;
  int64_t total = 0;
  for (const int t : tiles) costs.push_back(t + kUnitCost), total += t + kUnitCost;
  int64_t best = estimate(costs, hkv, W);
  if (best <= total * hkv / W + kUnitCost + kPartCost + kJoinCost) return Cut{0, 0};
  best = best * 19 / 20;                         // (less is not worth the partials' traffic)
  std::vector<int> sorted = tiles;
  std::sort(sorted.begin(), sorted.end(), std::greater<int>());
  Cut cut{0, 0};
  for (const int64_t whole : {int64_t(0), n * hkv / W * W / hkv}) {
    if (whole > 0 && whole >= n) continue;
    for (const int k : {2, 3, 4, 6, 8, 12, 16}) {
      const int longest = std::max(kMinPiece, (sorted[whole] + k - 1) / k);
      costs.clear();
      for (int64_t i = 0; i < n; ++i) {
        const int t = sorted[i], pieces = i < whole ? 1 : std::max(1, (t + longest - 1) / longest);
        for (int j = 0; j < pieces; ++j)
          costs.push_back((t + pieces - 1) / pieces + kUnitCost + (pieces > 1 ? kPartCost : 0));
      }
      const int64_t time = estimate(costs, hkv, W) + kJoinCost;
      if (time < best) {
        best = time;
        cut = Cut{whole, longest};
      }
    }
    if (n * hkv < W) break;
  }
  return cut;
}

int prompt_plan(const int32_t* qo_indptr, const int32_t* kv_indptr, int32_t batch, int32_t hq,
                int32_t hkv, int32_t head_dim, int32_t causal, kvc_prompt_schedule* sched,
                int32_t* plan_host, int64_t plan_capacity) {
  KVC_REQUIRE(sched, KVC_ERR_INVALID_ARG, "null schedule");
  KVC_REQUIRE(batch >= 0, KVC_ERR_INVALID_ARG, "negative batch");
  KVC_REQUIRE(batch == 0 || (qo_indptr && kv_indptr), KVC_ERR_INVALID_ARG, "null indptr");
  KVC_REQUIRE(hkv > 0 && hq > 0 && hq % hkv == 0, KVC_ERR_INVALID_ARG,
              "num_qo_heads must be a positive multiple of num_kv_heads");
  const int group = hq / hkv;
  KVC_REQUIRE((head_dim == 64 || head_dim == 128 || head_dim == 256) && group <= kMaxGroup,
              KVC_ERR_UNSUPPORTED,
              "prompt attention supports head_dim 64, 128, 256 and groups up to 128");
  const int tile_tokens = tile_rows(head_dim) / group, per_tile = tile_keys(head_dim);
  std::vector<int32_t> rec;
  int max_tiles = 0;
  int64_t end_q = 0, end_kv = 0, items = 0;
  for (int b = 0; b < batch; ++b) {
    const int64_t q_len = int64_t(qo_indptr[b + 1]) - qo_indptr[b];
    const int64_t kv_len = int64_t(kv_indptr[b + 1]) - kv_indptr[b];
    KVC_REQUIRE(q_len >= 0 && kv_len >= 0 && qo_indptr[b] >= 0 && kv_indptr[b] >= 0,
                KVC_ERR_INVALID_ARG, "qo_indptr and kv_indptr must be non-negative and "
                                     "non-decreasing");
    KVC_REQUIRE(kv_len < (int64_t(1) << 30) && q_len < (int64_t(1) << 30), KVC_ERR_INVALID_ARG,
                "sequence too long");
    items += (q_len + tile_tokens - 1) / tile_tokens;
    KVC_REQUIRE(items * hkv < (int64_t(1) << 27), KVC_ERR_INVALID_ARG,
                "too many (query tile, KV head) units");
    end_q = qo_indptr[b + 1];
    end_kv = kv_indptr[b + 1];
    for (int64_t t0 = 0; t0 < q_len; t0 += tile_tokens) {
      const int64_t last = std::min<int64_t>(t0 + tile_tokens, q_len) - 1;
      int64_t keys = causal ? last + kv_len - q_len + 1 : kv_len;
      keys = std::max<int64_t>(0, std::min<int64_t>(keys, kv_len));
      const int tiles = int((keys + per_tile - 1) / per_tile);
      max_tiles = std::max(max_tiles, tiles);
      const int32_t r8[kUnitInts] = {b, int32_t(t0), int32_t(q_len), int32_t(kv_len),
                                     qo_indptr[b], kv_indptr[b], tiles, 0};
      rec.insert(rec.end(), r8, r8 + kUnitInts);
    }
  }
  // Pieces in place of the items that are cut; joins: (first query, q_len, q offset,
  // first partial, pieces) of one head.
  std::vector<int> tiles;
  for (size_t i = 0; i < rec.size(); i += kUnitInts) tiles.push_back(rec[i + 6]);
  const Cut cut = choose_cut(tiles, hkv);
  std::vector<std::array<int32_t, 5>> joins;
  int parts = 0;
  if (cut.longest > 0) {
    // The longest `whole` items stay: those over `bar` tiles, and the first ones of them.
    std::sort(tiles.begin(), tiles.end(), std::greater<int>());
    const int bar = cut.whole > 0 ? tiles[cut.whole - 1] : INT32_MAX;
    int64_t at_bar = cut.whole > 0 ? cut.whole - (std::lower_bound(tiles.begin(), tiles.end(), bar,
                                                                  std::greater<int>()) -
                                                 tiles.begin())
                                   : 0;
    std::vector<int32_t> cut_rec;
    max_tiles = 0;
    for (size_t i = 0; i < rec.size(); i += kUnitInts) {
      const int32_t* r = rec.data() + i;
      const int t = r[6];
      const bool stays = t > bar || (t == bar && at_bar-- > 0);
      const int pieces = stays ? 1 : std::max(1, (t + cut.longest - 1) / cut.longest);
      if (pieces > 1) joins.push_back({r[1], r[2], r[4], parts, pieces});
      for (int j = 0; j < pieces; ++j) {
        const int from = int(int64_t(t) * j / pieces), to = int(int64_t(t) * (j + 1) / pieces);
        const int32_t r8[kUnitInts] = {r[0], r[1], r[2], r[3] - from * per_tile, r[4],
                                       r[5] + from * per_tile, to - from, pieces > 1 ? ++parts : 0};
        cut_rec.insert(cut_rec.end(), r8, r8 + kUnitInts);
        max_tiles = std::max(max_tiles, to - from);
      }
    }
    rec = std::move(cut_rec);
  }
  const int64_t n = int64_t(rec.size()) / kUnitInts;
  const int64_t W = plan_workgroups(n * hkv);
  sched->batch = batch;
  sched->num_qo_heads = hq;
  sched->num_kv_heads = hkv;
  sched->head_dim = head_dim;
  sched->causal = causal ? 1 : 0;
  sched->tile_tokens = tile_tokens;
  sched->num_units = int32_t(n * hkv);
  sched->num_workgroups = int32_t(W);
  sched->total_q = int32_t(end_q);
  sched->total_kv = int32_t(end_kv);
  sched->max_key_tiles = max_tiles;
  sched->num_joins = int32_t(joins.size()) * hkv;
  sched->num_parts = int64_t(parts) * hkv;
  sched->plan_ints = prompt_plan_ints(*sched);
  sched->workspace_bytes = prompt_workspace_bytes(*sched);
  KVC_REQUIRE(plan_capacity >= sched->plan_ints && (plan_host || sched->plan_ints == 0),
              KVC_ERR_WORKSPACE,
              "plan buffer too small: need " + std::to_string(sched->plan_ints) + " int32");
  if (n > 0) write_plan(rec, n, hkv, W, parts, plan_host);
  int32_t* dst = plan_host + sched->plan_ints - int64_t(sched->num_joins) * kJoinInts;
  for (int h = 0; h < hkv; ++h)
    for (const auto& j : joins) {
      const int32_t r8[kJoinInts] = {h, j[0], j[1], j[2], j[3] + h * parts, j[4], 0, 0};
      dst = std::copy_n(r8, kJoinInts, dst);
    }
  return ok();
}

template <typename T>
void launch(const PromptArgs& a, int head_dim, unsigned workgroups, hipStream_t s) {
  const dim3 grid(workgroups), block(unsigned(64 * kWaves(head_dim)));
  if (head_dim == 64) prompt_kernel<T, 64><<<grid, block, 0, s>>>(a);
  else if (head_dim == 128) prompt_kernel<T, 128><<<grid, block, 0, s>>>(a);
  else prompt_wide_kernel<T, 256><<<grid, block, 0, s>>>(a);
}

template <typename T>
void launch_join(const PromptArgs& a, int head_dim, const int4* joins, unsigned n, hipStream_t s) {
  const int rows = tile_rows(head_dim);
  const dim3 grid{n, unsigned(rows * head_dim / 1024)};
  if (head_dim == 64) prompt_join_kernel<T, 64><<<grid, 256, 0, s>>>(a, joins, rows);
  else if (head_dim == 128) prompt_join_kernel<T, 128><<<grid, 256, 0, s>>>(a, joins, rows);
  else prompt_join_kernel<T, 256><<<grid, 256, 0, s>>>(a, joins, rows);
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_prompt_plan(const int32_t* qo_indptr_host, const int32_t* kv_indptr_host,
                               int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                               int32_t head_dim, int32_t causal, kvc_prompt_schedule* schedule,
                               int32_t* plan_host, int64_t plan_capacity) {
  KVC_NO_THROW(return prompt_plan(qo_indptr_host, kv_indptr_host, batch, num_qo_heads,
                                  num_kv_heads, head_dim, causal, schedule, plan_host,
                                  plan_capacity));
}

extern "C" int kvc_prompt_run(const kvc_prompt_schedule* sched, const int32_t* plan,
                              void* workspace, int64_t workspace_bytes, const void* q,
                              int64_t q_token_stride, const void* key,
                              int64_t key_token_stride, const void* value,
                              int64_t value_token_stride, int32_t dtype, float sm_scale,
                              void* out, int64_t out_token_stride, float* lse, void* stream) {
  KVC_REQUIRE(sched, KVC_ERR_INVALID_ARG, "null schedule");
  const int Hq = sched->num_qo_heads, Hkv = sched->num_kv_heads, D = sched->head_dim;
  KVC_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= kMaxGroup &&
                  (D == 64 || D == 128 || D == 256) && sched->num_units >= 0 &&
                  sched->tile_tokens == tile_rows(D) / (Hq / Hkv) &&
                  sched->num_workgroups == plan_workgroups(sched->num_units) &&
                  sched->num_joins >= 0 && sched->num_parts >= 0 &&
                  sched->num_parts <= sched->num_units &&
                  sched->plan_ints == prompt_plan_ints(*sched) &&
                  sched->workspace_bytes == prompt_workspace_bytes(*sched),
              KVC_ERR_INVALID_ARG, "schedule not produced by kvc_prompt_plan");
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");
  KVC_REQUIRE(sm_scale > 0.f && std::isfinite(sm_scale), KVC_ERR_INVALID_ARG,
              "sm_scale must be positive and finite");
  if (sched->num_units == 0) return ok();
  KVC_REQUIRE(plan && q && out && (sched->total_kv == 0 || (key && value)), KVC_ERR_INVALID_ARG,
              "null pointer");
  const int64_t qw = int64_t(Hq) * D, kw = int64_t(Hkv) * D;
  KVC_REQUIRE(q_token_stride >= qw && out_token_stride >= qw && key_token_stride >= kw &&
                  value_token_stride >= kw,
              KVC_ERR_INVALID_ARG, "token stride smaller than the token's heads");
  // (a tile's tokens are addressed by 32-bit byte offsets)
  KVC_REQUIRE(q_token_stride < (int64_t(1) << 22) && key_token_stride < (int64_t(1) << 22) &&
                  value_token_stride < (int64_t(1) << 22) && out_token_stride < (int64_t(1) << 22),
              KVC_ERR_INVALID_ARG, "q, key, value or out tokens 8 MiB or more apart");
  KVC_REQUIRE(aligned(q, 16) && aligned(key, 16) && aligned(value, 16) && aligned(out, 16) &&
                  aligned(plan, 16) && q_token_stride % 8 == 0 && key_token_stride % 8 == 0 &&
                  value_token_stride % 8 == 0 && out_token_stride % 8 == 0,
              KVC_ERR_ALIGNMENT,
              "q/key/value/out/plan must be 16-byte aligned and token strides multiples of 8");
  KVC_REQUIRE(sched->num_parts == 0 || (workspace && workspace_bytes >= sched->workspace_bytes),
              KVC_ERR_WORKSPACE,
              "workspace too small: need " + std::to_string(sched->workspace_bytes) + " bytes");
  KVC_REQUIRE(aligned(workspace, 16), KVC_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  PromptArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(key);
  a.v = static_cast<const uint16_t*>(value);
  a.q_stride = q_token_stride;
  a.k_stride = key_token_stride;
  a.v_stride = value_token_stride;
  a.wg_units = reinterpret_cast<const int2*>(plan);
  a.units = reinterpret_cast<const int4*>(plan + table_ints(sched->num_workgroups));
  a.num_kv_heads = Hkv;
  a.group = Hq / Hkv;
  a.tile_tokens = sched->tile_tokens;
  a.causal = sched->causal;
  a.inv_group = (65536u + unsigned(a.group) - 1) / unsigned(a.group);
  a.scale_log2 = sm_scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_token_stride;
  a.lse = lse;
  a.parts = static_cast<float*>(workspace);
  a.part_max = a.parts + sched->num_parts * tile_rows(D) * D;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == KVC_DTYPE_BF16) launch<Bf16>(a, D, unsigned(sched->num_workgroups), s);
  else launch<Fp16>(a, D, unsigned(sched->num_workgroups), s);
  KVC_LAUNCH_CHECK();
  if (sched->num_joins > 0) {
    const int4* joins = reinterpret_cast<const int4*>(plan + sched->plan_ints -
                                                      int64_t(sched->num_joins) * kJoinInts);
    if (dtype == KVC_DTYPE_BF16) launch_join<Bf16>(a, D, joins, unsigned(sched->num_joins), s);
    else launch_join<Fp16>(a, D, joins, unsigned(sched->num_joins), s);
    KVC_LAUNCH_CHECK();
  }
  return ok();
}
