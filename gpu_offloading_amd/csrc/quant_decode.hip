// Decode attention over the quantised cache (quant.h, quant_cache.hip): request b's one
// query token against the tokens of pages indices[indptr[b] .. indptr[b+1]),
//   x_t = scale * ks_t * (q . kc_t),   out = sum_t softmax(x)_t * vs_t * vc_t,
// with codes kc, vc and their rows' scales ks, vs.
//
// What bounds it: every code is read once and used by the `group` query heads of its KV
// head, 4 * group flop per byte of codes, so HBM.  The products run on MFMA 16x16x32 with
// the query heads as one side (group <= 16, the rest zero), which leaves the VALU the
// conversion of the codes.
//
// A wave takes 32 tokens (two pages) of one KV head at a time, K and V straight from
// memory into registers, no LDS:
//   S^T = K Q^T   A: lane (t = l % 16, g = l / 16) holds pieces of token t's row, B: the same
//                 pieces of query row l % 16 (the order of the summed dims is free).  It
//                 leaves lane l with the scores of query row l % 16, tokens 4 g .. 4 g + 3.
//   O^T = V^T P^T B: those very scores, exponentiated, of both pages; A: lane (c = l % 16, g)
//                 holds dims c D/16 .. of tokens 4 g .. 4 g + 3, four bytes of four tokens
//                 transposed with byte permutes.  So the weights never change lanes.
// A row's running maximum is only raised (and O rescaled) where a score exceeds it by 2^8:
// the maximum needs no cross-lane step per tile.
//
// Split: the batch's pages, laid end to end, are cut into equal segments, one per
// workgroup and KV head; each finds its first request in indptr by itself.  The launch
// depends on the batch size alone, so a captured one serves other lengths and pages.  The
// part of a request in one segment is a piece; one that is a whole request is written out,
// the others leave (m, l, O) in the workspace, joined by quant_merge_kernel.
#include "quant.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace kvc {
namespace {

constexpr int kWaves = 4;             // waves of a workgroup
constexpr int kMinPages = 16;         // of a segment
constexpr float kRaise = 8.f;         // log2: how far a score may exceed the running maximum
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

struct QuantDecodeArgs {
  const uint16_t* q;
  int64_t q_stride;          // elements between requests
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* scales;
  int64_t block_stride;      // codes between blocks
  int64_t scales_stride;     // floats between blocks
  int64_t num_blocks;
  const int32_t* indptr;
  const int32_t* indices;
  int64_t num_indices;
  const int32_t* last_page_len;
  int32_t batch, hq, hkv, group;
  int32_t segments;          // per KV head
  float scale_log2;
  float* parts;              // [hkv][segments][2][group][D + 2]: m, l, O
  uint16_t* out;
  int64_t out_stride;        // elements between requests
  float* lse;                // may be null
};

// Pages per segment; the kernels agree on it.
__device__ __forceinline__ int segment_pages(const QuantDecodeArgs& a, int total) {
  return max(kMinPages, int((int64_t(total) + a.segments - 1) / a.segments));
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <bool kHalf>
__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (kHalf)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Sum or maximum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
template <typename F>
__device__ __forceinline__ float across(float v, F f) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const uint32_t w = __float_as_uint(v);
  const auto s = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// First request whose pages reach past `page` (pages counted from indptr[0]); the last one
// if none does.  64 entries of indptr are compared at a time.
__device__ __forceinline__ int find_request(const int32_t* indptr, int batch, int base, int page) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = batch;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = min((lane + 1) * step, n);
    // requests before the one looked for end at or below `page`
    const bool below = lane * step < n && indptr[lo + i] - base <= page;
    const int c = __popcll(__ballot(below));
    lo = uniform(min(lo + c * step, lo + n - 1));
    n = min(step, batch - lo);
    if (step == 1) break;
  }
  return lo;
}

template <int D>
struct VWord;
template <>
struct VWord<64> { using type = uint32_t; };
template <>
struct VWord<128> { using type = u32x2_t; };
template <>
struct VWord<256> { using type = u32x4_t; };

template <int D>
__device__ __forceinline__ uint32_t word(typename VWord<D>::type v, int i) {
  if constexpr (D == 64)
    return v;
  else
    return v[i];
}

template <int D, int kCode, bool kHalf>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 2 : 4) void quant_decode_kernel(
    QuantDecodeArgs a) {
  using V = typename VWord<D>::type;
  constexpr int kKLoads = D / 64;   // 16-byte pieces of a K row per lane
  constexpr int kDims = D / 16;     // dims of a V row per lane
  extern __shared__ float lds[];    // [kWaves][group][D + 4]: m, l, -, -, O
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  const uint32_t k_lane = row * D + g * 16, v_lane = g * 4 * D + row * kDims, s_lane = g * 16;
  const int head = blockIdx.x % a.hkv, segment = blockIdx.x / a.hkv;
  const int base = a.indptr[0], total = a.indptr[a.batch] - base;
  const int pages = segment_pages(a, total);
  const int group = a.group;
  float* const out_lse = a.lse;

  // Requests without tokens: zeros, and -inf.
  for (int b = segment; b < a.batch; b += a.segments) {
    if (a.indptr[b + 1] > a.indptr[b]) continue;
    for (int i = threadIdx.x; i < group * D; i += kWaves * 64)
      a.out[b * a.out_stride + int64_t(head) * group * D + i] = 0;
    if (out_lse && threadIdx.x < group)
      out_lse[int64_t(b) * a.hq + head * group + threadIdx.x] = -INFINITY;
  }
  int64_t at64 = int64_t(segment) * pages;
  if (at64 >= total) return;
  int at = int(at64);
  const int end = int(min(at64 + pages, int64_t(total)));
  int b = find_request(a.indptr, a.batch, base, at);

  while (at < end) {
    int first = a.indptr[b] - base, last = a.indptr[b + 1] - base;
    while (b < a.batch - 1 && last <= at) {
      first = last;
      last = a.indptr[++b + 1] - base;
    }
    if (last <= at) break;   // (an indptr that goes down)
    const int stop = min(last, end);
    const int tail = min(max(a.last_page_len[b], 0), kQuantPage);

    // The query rows of the head's group, as the B operand.
    uint4 q[kKLoads][2];
    const uint16_t* qp = a.q + b * a.q_stride + (int64_t(head) * group + min(row, group - 1)) * D;
#pragma unroll
    for (int j = 0; j < kKLoads; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q[j][h] = *reinterpret_cast<const uint4*>(qp + j * 64 + g * 16 + h * 8);
        if (row >= group) q[j][h] = make_uint4(0, 0, 0, 0);
      }

    float m = kLowest, l = 0.f;
    f32x4_t o[kDims] = {};
    for (int p = at + 2 * wave; p < stop; p += 2 * kWaves) {
      u32x4_t k[2][kKLoads];
      V v[2][4];
      f32x4_t ks[2], vs[2];
      int count[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t slot = int64_t(base) + p + i;
        int id = p + i < stop && slot >= 0 && slot < a.num_indices ? a.indices[slot] : -1;
        const bool held = id >= 0 && id < a.num_blocks;
        count[i] = uniform(!held ? 0 : p + i == last - 1 ? tail : kQuantPage);
        id = uniform(held ? id : 0);
        // (a uniform base and the lane's fixed 32-bit offset: no address arithmetic in VGPRs)
        const int64_t tile = int64_t(id) * a.block_stride + int64_t(head) * (kQuantPage * D);
        const uint8_t* kp = a.k_cache + tile;
#pragma unroll
        for (int j = 0; j < kKLoads; ++j)
          k[i][j] = __builtin_nontemporal_load(
              reinterpret_cast<const u32x4_t*>(kp + (k_lane + uint32_t(j * 64))));
        const uint8_t* vp = a.v_cache + tile;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[i][j] = __builtin_nontemporal_load(
              reinterpret_cast<const V*>(vp + (v_lane + uint32_t(j * D))));
        const uint8_t* sp = reinterpret_cast<const uint8_t*>(
            a.scales + int64_t(id) * a.scales_stride + head * (2 * kQuantPage));
        ks[i] = *reinterpret_cast<const f32x4_t*>(sp + s_lane);
        vs[i] = *reinterpret_cast<const f32x4_t*>(sp + (s_lane + uint32_t(kQuantPage * 4)));
      }

      f32x4_t x[2] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kKLoads; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w0 = k[i][j][2 * h], w1 = k[i][j][2 * h + 1];
            x[i] = mfma<kHalf>(make_uint4(decode2<kCode, kHalf, 0>(w0), decode2<kCode, kHalf, 1>(w0),
                                          decode2<kCode, kHalf, 0>(w1), decode2<kCode, kHalf, 1>(w1)),
                               q[j][h], x[i]);
          }
      float most = kLowest;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // One rounding per factor: the difference from the maximum is then exact where it counts.
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[i][j] = x[i][j] * ks[i][j] * a.scale_log2;
          if (count[i] < kQuantPage && g * 4 + j >= count[i]) x[i][j] = -INFINITY;
          most = fmaxf(most, x[i][j]);
        }
      }
      if (__any(most > m + kRaise)) {
        const float top = fmaxf(m, across(most, [](float s, float t) { return fmaxf(s, t); }));
        const float f = fast_exp2(m - top);
        l *= f;
#pragma unroll
        for (int e = 0; e < kDims; ++e) o[e] *= f;
        m = top;
      }
      // Weights: exact to fp32 in l; for the products they carry the V rows' scales and are
      // bf16 (2^-9 of each weight, below an output's own bf16 step), for fp16 outputs a
      // pair of bf16 (2^-17): fp16 itself has no room for any scale.
      float w[8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = fast_exp2(x[i][j] - m);
          l += e;
          w[i * 4 + j] = e * vs[i][j];
        }
      if (count[0] < kQuantPage || count[1] < kQuantPage) {
        // What masked slots hold (codes that are NaN, scales that are anything) does not enter.
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (g * 4 + j >= count[i]) {
              w[i * 4 + j] = 0.f;
              v[i][j] = V{};
            }
      }
      uint4 hi, lo;
      hi.x = pack2<false>(w[0], w[1]);
      hi.y = pack2<false>(w[2], w[3]);
      hi.z = pack2<false>(w[4], w[5]);
      hi.w = pack2<false>(w[6], w[7]);
      if constexpr (kHalf) {
        lo.x = pack2<false>(w[0] - bf16lo(hi.x), w[1] - bf16hi(hi.x));
        lo.y = pack2<false>(w[2] - bf16lo(hi.y), w[3] - bf16hi(hi.y));
        lo.z = pack2<false>(w[4] - bf16lo(hi.z), w[5] - bf16hi(hi.z));
        lo.w = pack2<false>(w[6] - bf16lo(hi.w), w[7] - bf16hi(hi.w));
      }
#pragma unroll
      for (int e4 = 0; e4 < kDims / 4; ++e4) {
        // bytes e of four tokens -> one word per dim
        uint32_t t[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t r0 = word<D>(v[i][0], e4), r1 = word<D>(v[i][1], e4);
          const uint32_t r2 = word<D>(v[i][2], e4), r3 = word<D>(v[i][3], e4);
          const uint32_t a01 = __builtin_amdgcn_perm(r1, r0, 0x05010400u);   // r0.0 r1.0 r0.1 r1.1
          const uint32_t a23 = __builtin_amdgcn_perm(r3, r2, 0x05010400u);
          const uint32_t b01 = __builtin_amdgcn_perm(r1, r0, 0x07030602u);   // r0.2 r1.2 r0.3 r1.3
          const uint32_t b23 = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
          t[i][0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
          t[i][1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
          t[i][2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
          t[i][3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint4 vt = make_uint4(
              decode2<kCode, false, 0>(t[0][e]), decode2<kCode, false, 1>(t[0][e]),
              decode2<kCode, false, 0>(t[1][e]), decode2<kCode, false, 1>(t[1][e]));
          o[e4 * 4 + e] = mfma<false>(vt, hi, o[e4 * 4 + e]);
          if constexpr (kHalf) o[e4 * 4 + e] = mfma<false>(vt, lo, o[e4 * 4 + e]);
        }
      }
    }

    // The waves' parts of the piece, joined in LDS.
    l = across(l, [](float s, float t) { return s + t; });
    if (row < group) {
      float* to = lds + (wave * group + row) * (D + 4);
      if (g == 0) {
        to[0] = m;
        to[1] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < kDims; e += 4)
          *reinterpret_cast<f32x4_t*>(to + 4 + (g * 4 + i) * kDims + e) =
              f32x4_t{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
    }
    __syncthreads();
    const bool whole = first >= at && last <= end;
    float* part = a.parts + ((int64_t(head) * a.segments + segment) * 2 + (first > at64 ? 1 : 0)) *
                                (int64_t(group) * (D + 2));
    for (int i = threadIdx.x; i < group * (D / 4); i += kWaves * 64) {
      const int r = i / (D / 4), c = i % (D / 4);
      float top = kLowest, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, lds[(w * group + r) * (D + 4)]);
      f32x4_t acc = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float* from = lds + (w * group + r) * (D + 4);
        const float f = fast_exp2(from[0] - top);
        sum += from[1] * f;
        acc += *reinterpret_cast<const f32x4_t*>(from + 4 + c * 4) * f;
      }
      if (whole) {
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        uint2 packed;
        packed.x = pack2<kHalf>(acc[0] * f, acc[1] * f);
        packed.y = pack2<kHalf>(acc[2] * f, acc[3] * f);
        *reinterpret_cast<uint2*>(a.out + b * a.out_stride + (int64_t(head) * group + r) * D + c * 4) =
            packed;
        if (out_lse && c == 0)
          out_lse[int64_t(b) * a.hq + head * group + r] =
              sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
      } else {
        float* to = part + r * (D + 2);
        if (c == 0) {
          to[0] = top;
          to[1] = sum;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) to[2 + c * 4 + e] = acc[e];
      }
    }
    __syncthreads();
    at = stop;
  }
}

// Joins the pieces of one request and query head.
template <int D, bool kHalf>
__global__ __launch_bounds__(D) void quant_merge_kernel(QuantDecodeArgs a) {
  const int b = blockIdx.y, hq = blockIdx.x;
  const int base = a.indptr[0], total = a.indptr[a.batch] - base;
  const int first = a.indptr[b] - base, last = a.indptr[b + 1] - base;
  const int pages = segment_pages(a, total);
  if (first < 0 || last <= first || last > total) return;
  const int s0 = first / pages, s1 = (last - 1) / pages;
  if (s0 == s1) return;
  const int head = hq / a.group, r = hq % a.group;
  const int64_t step = int64_t(a.group) * (D + 2);
  const float* p0 = a.parts + (int64_t(head) * a.segments + s0) * 2 * step + r * (D + 2) +
                    (first > s0 * pages ? step : 0);
  const float* ps = a.parts + (int64_t(head) * a.segments) * 2 * step + r * (D + 2);
  float top = p0[0];
  for (int s = s0 + 1; s <= s1; ++s) top = fmaxf(top, ps[s * 2 * step]);
  float f = fast_exp2(p0[0] - top), sum = p0[1] * f, acc = p0[2 + threadIdx.x] * f;
  for (int s = s0 + 1; s <= s1; ++s) {
    const float* p = ps + s * 2 * step;
    f = fast_exp2(p[0] - top);
    sum += p[1] * f;
    acc += p[2 + threadIdx.x] * f;
  }
  const float y = sum == 0.f ? 0.f : acc / sum;
  a.out[b * a.out_stride + int64_t(hq) * D + threadIdx.x] = uint16_t(pack2<kHalf>(y, y));
  if (a.lse && threadIdx.x == 0)
    a.lse[int64_t(b) * a.hq + hq] = sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
}

// Segments per KV head: the workgroups that the GPU holds at once, over the heads.
int segments_of(int hkv, int head_dim) {
  const int held = 256 * (head_dim == 256 ? 2 : 4);
  return std::max(1, held / hkv);
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int64_t kvc_quantized_decode_workspace_bytes(int32_t batch, int32_t num_qo_heads,
                                                        int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
  return int64_t(segments_of(num_kv_heads, head_dim)) * 2 * num_qo_heads * (head_dim + 2) * 4;
}

extern "C" int kvc_quantized_decode(
    const void* q, int64_t q_batch_stride, const void* key_cache, const void* value_cache,
    const float* scales, int64_t cache_block_stride, int64_t scales_block_stride,
    int64_t num_blocks, const int32_t* indptr, const int32_t* indices, int64_t num_indices,
    const int32_t* last_page_len, int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t page_size, int32_t dtype, int32_t code, float sm_scale,
    void* workspace, int64_t workspace_bytes, void* out, int64_t out_batch_stride, float* lse,
    void* stream) {
  KVC_REQUIRE(batch >= 0 && num_indices >= 0, KVC_ERR_INVALID_ARG, "negative batch or num_indices");
  if (batch == 0) return ok();
  KVC_REQUIRE(q && key_cache && value_cache && scales && indptr && last_page_len && out &&
                  (indices || num_indices == 0),
              KVC_ERR_INVALID_ARG, "null pointer");
  KVC_REQUIRE(batch <= 65535, KVC_ERR_INVALID_ARG, "batch > 65535");
  KVC_REQUIRE(code == KVC_CODE_E4M3 || code == KVC_CODE_INT8, KVC_ERR_UNSUPPORTED,
              "code must be KVC_CODE_E4M3 or KVC_CODE_INT8");
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");
  KVC_REQUIRE(num_kv_heads > 0 && num_qo_heads > 0 && num_qo_heads % num_kv_heads == 0 &&
                  num_kv_heads <= 65535 && num_blocks > 0,
              KVC_ERR_INVALID_ARG, "bad head counts or no blocks");
  const int group = num_qo_heads / num_kv_heads;
  KVC_REQUIRE(group <= 16, KVC_ERR_UNSUPPORTED, "at most 16 query heads per KV head");
  KVC_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, KVC_ERR_UNSUPPORTED,
              "head_dim must be 64, 128 or 256");
  KVC_REQUIRE(page_size == kQuantPage, KVC_ERR_UNSUPPORTED, "page_size must be 16");
  KVC_REQUIRE(sm_scale > 0.f && std::isfinite(sm_scale * kLog2e), KVC_ERR_INVALID_ARG,
              "sm_scale must be positive and finite");
  KVC_REQUIRE(cache_block_stride >= int64_t(num_kv_heads) * kQuantPage * head_dim &&
                  scales_block_stride >= int64_t(num_kv_heads) * 2 * kQuantPage,
              KVC_ERR_INVALID_ARG, "a block stride is smaller than a block");
  const int64_t row = int64_t(num_qo_heads) * head_dim;
  KVC_REQUIRE(q_batch_stride >= row && out_batch_stride >= row, KVC_ERR_INVALID_ARG,
              "q or out stride smaller than a request's heads");
  KVC_REQUIRE(aligned(key_cache, 16) && aligned(value_cache, 16) && aligned(scales, 16) &&
                  cache_block_stride % 16 == 0 && scales_block_stride % 4 == 0 && aligned(q, 16) &&
                  q_batch_stride % 8 == 0 && aligned(out, 8) && out_batch_stride % 4 == 0,
              KVC_ERR_ALIGNMENT,
              "q, the caches and the scales must be 16-byte aligned, out 8-byte, with strides alike");
  const int64_t need = kvc_quantized_decode_workspace_bytes(batch, num_qo_heads, num_kv_heads, head_dim);
  KVC_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16), KVC_ERR_WORKSPACE,
              "workspace too small or not 16-byte aligned");

  QuantDecodeArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_batch_stride;
  a.k_cache = static_cast<const uint8_t*>(key_cache);
  a.v_cache = static_cast<const uint8_t*>(value_cache);
  a.scales = scales;
  a.block_stride = cache_block_stride;
  a.scales_stride = scales_block_stride;
  a.num_blocks = num_blocks;
  a.indptr = indptr;
  a.indices = indices;
  a.num_indices = num_indices;
  a.last_page_len = last_page_len;
  a.batch = batch;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.group = group;
  a.segments = segments_of(num_kv_heads, head_dim);
  a.scale_log2 = sm_scale * kLog2e;
  a.parts = static_cast<float*>(workspace);
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_batch_stride;
  a.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = unsigned(a.segments) * unsigned(num_kv_heads);
  const unsigned lds = unsigned(kWaves * group * (head_dim + 4) * 4);

  auto launch = [&](auto d, auto c, auto half) {
    constexpr int D = decltype(d)::value, C = decltype(c)::value;
    constexpr bool H = decltype(half)::value;
    auto* kernel = &quant_decode_kernel<D, C, H>;
    if (lds > 65536)
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
    kernel<<<grid, kWaves * 64, lds, s>>>(a);
    quant_merge_kernel<D, H><<<dim3(unsigned(num_qo_heads), unsigned(batch)), D, 0, s>>>(a);
  };
  auto by_type = [&](auto d, auto c) {
    if (dtype == KVC_DTYPE_FP16)
      launch(d, c, std::true_type{});
    else
      launch(d, c, std::false_type{});
  };
  auto by_code = [&](auto d) {
    if (code == KVC_CODE_INT8)
      by_type(d, std::integral_constant<int, KVC_CODE_INT8>{});
    else
      by_type(d, std::integral_constant<int, KVC_CODE_E4M3>{});
  };
  if (head_dim == 64)
    by_code(std::integral_constant<int, 64>{});
  else if (head_dim == 128)
    by_code(std::integral_constant<int, 128>{});
  else
    by_code(std::integral_constant<int, 256>{});
  KVC_LAUNCH_CHECK();
  return ok();
}
