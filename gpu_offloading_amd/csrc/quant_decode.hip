// Decode attention over the quantised cache (quant.h, quant_cache.hip): request b's one
// query token against the tokens of pages indices[indptr[b] .. indptr[b+1]),
//   x_t = scale * ks_t * (q . kc_t),   out = sum_t softmax(x)_t * vs_t * vc_t,
// with codes kc, vc and their rows' scales ks, vs.
//
// What bounds it: every code is read once and used by the `group` query heads of its KV
// head, 2 * group flop per byte of codes, so HBM.  The products run on MFMA 16x16x32 with
// the query heads as one side (group <= 16), which leaves the VALU the conversion of the codes.
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
// K, V and scales are loaded a tile ahead, each part into the registers that the tile at hand has
// just freed; page ids and lengths go through the scalar cache.
//
// Split, decided on the device from indptr (so a captured launch serves other lengths and pages):
//   cut        the batch's requests, laid end to end, are cut into segments of equal work, one per
//              workgroup and KV head; each finds its first request in indptr by itself.  The part of
//              a request in a segment is a piece, whose tiles the workgroup's waves take in turn and
//              join in LDS (a very short request is a wave's).  A piece that is a whole request is
//              written out; the others leave (m, l, O) in the workspace, which quant_merge_kernel joins.
//   workgroup  each request is a workgroup's (per KV head) where none is long,
//   wave       or a wave's where they are many and short.
//
// 64 requests of 512 to 4096 tokens, 8 KV heads of 128, 4 query heads each: 54.0 us (the kernel 49.7, its
// join 4.6), 300 MB at 5.5 TB/s; 16 of 32767: 166 us (162), 6.7 TB/s, where the same loads alone take 161.
// Before the first loads lie 2.4 us: the launch, indptr, a page id.
#include "quant.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace kvc {
namespace {

constexpr int kWaves = 4;             // waves of a workgroup
constexpr int kScan = 4096;            // requests that are looked through for longer ones

// Waves per SIMD, which bounds their registers, ...
constexpr int per_simd(int head_dim) { return head_dim == 64 ? 4 : head_dim == 128 ? 3 : 2; }
// ... and workgroups per CU that a batch is cut for: these keep a tile per wave in flight, 34 KB per CU
// at head_dim 64 and 67 KB at 128 and 256, and more only compete (16 x 32767 tokens at head_dim 128:
// 166 us with 2, 169 with 3; 16 of 20000 to 32000 at head_dim 64: 79 with 2, 81 with 4) and leave
// more to join.
constexpr int cut_for(int head_dim) { return head_dim == 256 ? 1 : 2; }

constexpr float kRaise = 8.f;         // log2: how far a score may exceed the running maximum
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Division of numbers below 2^31 by one of 1 to 512, rounded down (one more for some above 2^23, which
// the segments can take).  An ordinary division here, in front of all loads, costs 0.2 us.
struct Divisor {
  uint64_t inverse;
  uint32_t by;
  explicit Divisor(uint32_t n = 1) : inverse(((uint64_t(1) << 32) + n - 1) / n), by(n) {}
};

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
  int32_t groups;            // workgroups per KV head, at least as many
  Divisor in_all, in_cus;    // by the segments, by the CUs per KV head
  int32_t even_from;         // units per segment from which all segments are used
  float scale_log2;
  float* parts;              // [hkv][segments][2][group][D + 4]: m, l, -, -, O
  uint16_t* out;
  int64_t out_stride;        // elements between requests
  float* lse;                // may be null
};

// Pages of the batch: what indptr spans, as far as there are indices (pages past them hold no tokens).
__device__ __forceinline__ int pages_in_all(const QuantDecodeArgs& a, int base, int end) {
  return max(int(min(int64_t(end) - base, a.num_indices - max(base, 0))), 0);
}

// Segments are equal in units: a page is one, and so are `each` in front of each request's pages, for the
// piece's start and end (about 3 us, eight pages' time).  Fewer where requests are short or missing, as
// empty ones count too: an eighth to a quarter of the pages in all for 8 to 64 pages per request, less for
// longer ones (2% at 512), and more only below 8 (as much as the pages at one per request).  None where
// they are so long that it does not matter: then segments may end with requests.  (100 requests of 10
// to 1100 tokens 32.0 -> 28.4 us, 64 of 100 to 1200 23.2 -> 22.3, 60 of 1 to 40 and 4 of 8000 24.1 -> 20.2;
// in another run at head_dim 64 22.0 -> 19.8, 18.0 -> 16.3, 19.2 -> 14.2, at 256 47.1 -> 44.2, 39.6 -> 36.4,
// 45.2 -> 28.3.)
__device__ __forceinline__ int each_of(int batch, int total) {
  const int64_t t = total, b = batch;
  return b == 1 || t >= b * 512 ? 0 : t >= b * 32 ? 8 : t >= b * 16 ? 4 : t >= b * 8 ? 2 : 1;
}

// Units per segment; the kernels agree on it.  Segments of few are one per CU, not one and a half, which leaves some CUs twice the others' work (one request of 8192 tokens, 8 KV heads: 9.0 us
// in 256 segments, 9.7 in 512, 10.7 in 344; 16 of 1000 to 5000, 2 KV heads: 14.5, 15.6 and 16.1).  Nor are
// they below one round of the waves, or two where requests would on average be in more pieces than the
// 64 that the join takes at a time (4 of 3000, 2 KV heads: 9.9 us with one round, 10.9 with two; one of
// 18000, 11.9 and 10.9).
__device__ __forceinline__ int segment_units(const QuantDecodeArgs& a, int all) {
  auto ceil_div = [&](Divisor d) {
    return int(uint64_t(uint32_t(all) + d.by - 1) * d.inverse >> 32);
  };
  const int even = ceil_div(a.in_all);
  if (even >= a.even_from) return even;
  const bool few = int64_t(all) <= int64_t(a.batch) * (64 * 2 * kWaves);
  return max(ceil_div(a.in_cus), (few ? 2 : 4) * kWaves);
}

// Index arrays are read through the scalar cache, ahead of use: a vector load of a page id
// would have to be waited for together with all the K and V loads in front of it.
typedef const int32_t __attribute__((address_space(4))) * ScalarInts;
__device__ __forceinline__ ScalarInts scalar_ints(const int32_t* p) {
  return (ScalarInts)reinterpret_cast<uintptr_t>(p);
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

// First request whose end reaches past a place (in pages from indptr[0], `each` more per request; the
// last one if none does), and its first page and the one behind its last.  64 entries of indptr are compared at a time; the
// first 64 are loaded before the page is known, beside what it depends on.
struct Search {
  int entry, step;

  __device__ __forceinline__ void start(const int32_t* indptr, int batch) {
    const int lane = threadIdx.x & 63;
    step = (batch + 63) / 64;
    entry = indptr[min((lane + 1) * step, batch)];
  }
  __device__ __forceinline__ int find(const int32_t* indptr, int batch, int base, int at, int each,
                                      int& first, int& last) const {
    const int lane = threadIdx.x & 63;
    // blocks of `step` requests before the one looked for end at or below `at`
    int c = __popcll(__ballot(lane * step < batch &&
                              entry - base + each * min((lane + 1) * step, batch) <= at));
    if (step == 1) {
      c = uniform(min(c, batch - 1));
      last = __builtin_amdgcn_readlane(entry, c) - base;
      first = c ? __builtin_amdgcn_readlane(entry, max(c - 1, 0)) - base : 0;
      return c;
    }
    int lo = uniform(min(c * step, batch - 1)), n = min(step, batch - lo);
    while (n > 1) {
      const int s = (n + 63) / 64;
      const int i = lo + min((lane + 1) * s, n);
      const int e = indptr[i];
      c = __popcll(__ballot(lane * s < n && e - base + each * i <= at));
      const int skip = min(c * s, n - 1);
      lo = uniform(lo + skip);
      n = s == 1 ? 1 : min(s, n - skip);
    }
    first = scalar_ints(indptr)[lo] - base;
    last = scalar_ints(indptr)[lo + 1] - base;
    return lo;
  }
};

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

// Whether no request has more pages than one workgroup streams in about the time that cutting
// and joining it costs: then each is a workgroup's (per KV head) and none is cut.  64 pages where the
// requests alone fill the GPU (64 requests of 600 to 1000 tokens, 8 KV heads: 26.0 cut, 23.5 us whole),
// 32 where they are few (one of 700: 7.6 and 9.2; 4 of 100 to 700: 10.0 and 10.9; 16 of 200 to 500, whole,
// 9.7, cut 11.2), else 48 (24 of 100 to 700: 13.8 and 11.5).  Every wave looks through
// indptr by itself, beside loads that it waits for anyway; batches too large for that are cut.
// (These figures are for 8 KV heads of 128.  The limits count pages, whatever a page weighs; cut and
// whole at 64: 24 of 100 to 700 11.5 and 9.4, 64 of 600 to 1000 17.2 and 14.6, 16 of 200 to 500 9.1 and
// 8.3; at 256: 16.5 and 14.8, 39.7 and 38.2, 12.3 and 11.8.  Left whole, and
// without the join's launch, somewhat longer ones would be faster at 64: 4 of 100 to 700 8.8 and 7.6.)
__host__ __device__ inline int whole_pages(int batch, int hkv) {
  return int64_t(batch) * hkv >= 256 ? 64 : batch <= 16 ? 32 : 48;
}
// Where the requests are more than the workgroups and shorter still, a wave takes one by itself: no
// round with idle waves, no join (256 requests of 10 to 180 tokens, 8 KV heads: 20.6 -> 17.5 us, of 16
// to 300 25.3 -> 23.7; but 64 of these, a workgroup each 11.3, a wave each 14.3, and 128 of up to 600
// tokens 21.6 and 23.7.  At head_dim 64 the four are 13.7 -> 11.7, 16.1 -> 14.7, 8.1 and 9.3, 13.8 and
// 18.0; at 256 32.3 -> 25.7, 39.4 -> 36.3, 12.6 and 13.6, 35.4 both).
enum class Share { cut, workgroup, wave };
constexpr int kWavePages = 20, kWaveRequests = 768;
// In a segment, whole requests of so few pages are a wave's each, too (300 requests of 1 to 16 tokens and one
// of 1100 31.1 -> 14.9 us, 1000 of 1 to 40 and 4 of 8000 104 -> 46; up to 8 or 20 pages a wave that has one
// holds up the others' next piece: 200 of 10 to 1500 63.8, 65.3 and 69.5; the first two at head_dim 64
// 24.9 -> 12.6 and 70.7 -> 33.6, at 256 38.2 -> 17.8 and 180.7 -> 77.7).
constexpr int kSoloPages = 4;
__device__ __forceinline__ Share share_of(const QuantDecodeArgs& a) {
  if (a.batch > kScan) return Share::cut;
  const int most = whole_pages(a.batch, a.hkv);
  const int listed = int(min(a.num_indices, int64_t(INT32_MAX)));
  int longest = 0;
  for (int i = threadIdx.x & 63; i < a.batch; i += 256) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = min(i + u * 64, a.batch - 1);
      longest = max(longest, min(a.indptr[j + 1], listed) - a.indptr[j]);
    }
  }
  if (__any(longest > most)) return Share::cut;
  return int64_t(a.batch) * a.hkv >= kWaveRequests && !__any(longest > kWavePages) ? Share::wave
                                                                                   : Share::workgroup;
}

// Barrier between the waves' uses of LDS.  (__syncthreads would also wait for the global loads.)
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Dims 4 c .. 4 c + 3 of a finished query row.
template <int D, bool kHalf>
__device__ __forceinline__ void write_out(const QuantDecodeArgs& a, int b, int hq, int c, float top,
                                          float sum, f32x4_t acc) {
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(a.out + b * a.out_stride + int64_t(hq) * D + c * 4) =
      make_uint2(pack2<kHalf>(acc[0] * f, acc[1] * f), pack2<kHalf>(acc[2] * f, acc[3] * f));
  if (a.lse && c == 0)
    a.lse[int64_t(b) * a.hq + hq] = sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
}

template <int D, int kCode, bool kHalf>
__global__ __launch_bounds__(kWaves * 64, per_simd(D)) void quant_decode_kernel(
    QuantDecodeArgs a) {
  using V = typename VWord<D>::type;
  constexpr int kKLoads = D / 64;   // 16-byte pieces of a K row per lane
  constexpr int kDims = D / 16;     // dims of a V row per lane
  extern __shared__ float lds[];    // [kWaves][group][D + 4]: m, l, -, -, O
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % a.hkv, segment = blockIdx.x / a.hkv;
  // K rows of 128 bytes and more are loaded as whole 128-byte lines, eight rows at a time: lane (t,
  // g) loads the piece 2 g + t / 8 of rows t % 8 and t % 8 + 8, and trades one of the two with lane
  // (t ^ 8, g).  (The same bytes in halves of lines: 6.5 TB/s of loads alone instead of 6.9.)
  const uint32_t k_lane = D == 64 ? row * D + g * 16 : (row & 7) * D + (g * 2 + (row >> 3)) * 16;
  const uint32_t v_lane = g * 4 * D + row * kDims, s_lane = g * 16;
  const ScalarInts indptr = scalar_ints(a.indptr), indices = scalar_ints(a.indices);
  const ScalarInts lengths = scalar_ints(a.last_page_len);
  Search search;
  search.start(a.indptr, a.batch);
  const int base = indptr[0], total = pages_in_all(a, base, indptr[a.batch]);
  const int each = each_of(a.batch, total), all = total + each * a.batch;
  const int units = segment_units(a, all);
  const int group = a.group;
  const Share share = share_of(a);
  const bool whole_requests = share != Share::cut, alone = share == Share::wave;
  if (!whole_requests && segment >= a.segments) return;
  const int64_t lo64 = int64_t(segment) * units;
  const int lo = int(min(lo64, int64_t(all))), hi = int(min(lo64 + units, int64_t(all)));

  // The query rows of the head's group, as the B operand.  (Rows past the group are copies
  // of its last: nothing reads what comes of them.)
  uint4 q[kKLoads][2];
  // Two pages per tile.  A tile's successor is loaded part by part as the registers fall free: K
  // after the scores, V after the products.  (Two sets of registers, all of the successor
  // ahead of the work, were no faster over long requests and leave room for fewer waves.)
  float m, l;
  f32x4_t o[kDims];
  u32x4_t k[2][kKLoads];
  V v[2][4];
  f32x4_t ks[2], vs[2];
  int count[2];              // tokens that a page holds
  int64_t id[2];
  int raw[2];                // the next tile's ids, as indices has them
  auto fetch = [&](int page) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      raw[i] = indices[max(min(int64_t(base) + page + i, a.num_indices - 1), int64_t(0))];
  };
  // Pages `page` and `page` + 1 of a piece that ends at `stop`, its request at `last`.
  auto place = [&](int (&n)[2], int page, int stop, int last, int tail) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool held = page + i < stop && raw[i] >= 0 && raw[i] < a.num_blocks;
      id[i] = held ? raw[i] : 0;
      n[i] = !held ? 0 : page + i == last - 1 ? tail : kQuantPage;
    }
  };
  // (a uniform base and the lane's fixed 32-bit offset: no address arithmetic in VGPRs)
  auto load_k = [&] {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* from = a.k_cache + id[i] * a.block_stride + int64_t(head) * (kQuantPage * D);
#pragma unroll
      for (int j = 0; j < kKLoads; ++j)
        k[i][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(
            from + (k_lane + uint32_t(j / 2 * 128 + j % 2 * 8 * D))));
    }
  };
  auto load_s = [&](f32x4_t (&to)[2], int kv) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* from = reinterpret_cast<const uint8_t*>(
          a.scales + id[i] * a.scales_stride + (head * 2 + kv) * kQuantPage);
      to[i] = *reinterpret_cast<const f32x4_t*>(from + s_lane);
    }
  };
  auto load_v = [&] {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* from = a.v_cache + id[i] * a.block_stride + int64_t(head) * (kQuantPage * D);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[i][j] = __builtin_nontemporal_load(
            reinterpret_cast<const V*>(from + (v_lane + uint32_t(j * D))));
    }
  };
  auto tile = [&](auto more) {
    constexpr bool kMore = decltype(more)::value;
    if constexpr (D > 64) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kKLoads; j += 2)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x0 = k[i][j][w], x1 = k[i][j + 1][w];
            k[i][j][w] = __builtin_amdgcn_update_dpp(x0, x1, kDppRowRor8, 0xF, 0xC, false);
            k[i][j + 1][w] = __builtin_amdgcn_update_dpp(x1, x0, kDppRowRor8, 0xF, 0x3, false);
          }
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
    if constexpr (kMore) load_k();
    // The scaled score is rounded before the maximum is taken from it: their difference is
    // never above the running maximum's by a rounding.
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = x[i][j] * ks[i][j] * a.scale_log2;
    if constexpr (kMore) load_s(ks, 0);
    const bool partial = count[0] < kQuantPage || count[1] < kQuantPage;
    if (partial) {
      // What masked slots hold (codes that are NaN, scales that are anything) does not enter.
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (g * 4 + j >= count[i]) {
            x[i][j] = -INFINITY;
            vs[i][j] = 0.f;
            v[i][j] = V{};
          }
    }
    float most = kLowest;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) most = fmaxf(most, x[i][j]);
    if (__any(most > m + kRaise)) {
      const float top = fmaxf(m, across(most, [](float s, float t) { return fmaxf(s, t); }));
      const float f = fast_exp2(m - top);
      l *= f;
#pragma unroll
      for (int e = 0; e < kDims; ++e) o[e] *= f;
      m = top;
    }
    // Weights: fp32 in l; for the products they carry the V rows' scales and are pairs of bf16, the
    // weight and what its rounding left (2^-16 of it).  One bf16 would be off by as much as a bf16
    // output's own rounding, fp16 has no room for any scale; the second product costs 0.5 to
    // 1.5% (64 requests of 512 to 4096 tokens 53.8 -> 54.0 us).
    float w[8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = fast_exp2(x[i][j] - m);
        l += e;
        w[i * 4 + j] = e * vs[i][j];
      }
    if constexpr (kMore) load_s(vs, 1);
    uint4 hi, lo;
    hi.x = pack2<false>(w[0], w[1]);
    hi.y = pack2<false>(w[2], w[3]);
    hi.z = pack2<false>(w[4], w[5]);
    hi.w = pack2<false>(w[6], w[7]);
    lo.x = pack2<false>(w[0] - bf16lo(hi.x), w[1] - bf16hi(hi.x));
    lo.y = pack2<false>(w[2] - bf16lo(hi.y), w[3] - bf16hi(hi.y));
    lo.z = pack2<false>(w[4] - bf16lo(hi.z), w[5] - bf16hi(hi.z));
    lo.w = pack2<false>(w[6] - bf16lo(hi.w), w[7] - bf16hi(hi.w));
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
        o[e4 * 4 + e] = mfma<false>(vt, lo, o[e4 * 4 + e]);
      }
    }
    if constexpr (kMore) load_v();
  };

  int first = 0, last = 0, b = alone ? segment * kWaves + wave : segment;
  const int stride = alone ? a.groups * kWaves : a.groups;
  if (!whole_requests) {
    if (lo < hi)
      b = search.find(a.indptr, a.batch, base, lo, each, first, last);
    else
      b = a.batch;
  }
  auto next = [&] {
    if (whole_requests) {
      b += stride;
      return;
    }
    first = last;
    if (++b < a.batch) last = indptr[b + 1] - base;
    if (last <= first && b < a.batch - 1) {   // (requests without pages)
      const int to = search.find(a.indptr, a.batch, base, first, 0, first, last);
      b = to > b ? to : a.batch;              // (never back, where an indptr goes down)
    }
  };
  for (; b < a.batch; next()) {
    int begin, end;
    if (whole_requests) {
      first = max(indptr[b] - base, 0);
      last = indptr[b + 1] - base;
      begin = first;
      end = min(last, total);
    } else {
      begin = lo - each * (b + 1);
      end = min(hi - each * (b + 1), total);
      if (first >= end) break;
    }
    const int at = max(max(first, begin), 0), stop = min(last, end);
    if (at >= stop) continue;
    const bool whole = first >= begin && min(last, total) <= end;
    const bool solo = alone || (!whole_requests && whole && stop - at <= kSoloPages);
    if (solo && !alone && b % kWaves != wave) continue;
    const int round = solo ? 2 : 2 * kWaves;   // pages that are taken at a time
    const int tail = min(max(lengths[b], 0), kQuantPage);
    m = kLowest;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < kDims; ++e) o[e] = f32x4_t{};

    int p = solo ? at : at + 2 * wave;
    if (p < stop) {
      fetch(p);
      const uint16_t* from =
          a.q + b * a.q_stride + (int64_t(head) * group + min(row, group - 1)) * D;
#pragma unroll
      for (int j = 0; j < kKLoads; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          q[j][h] = *reinterpret_cast<const uint4*>(
              from + (D == 64 ? g * 16 : j / 2 * 128 + g * 32 + j % 2 * 16) + h * 8);
      place(count, p, stop, last, tail);
      fetch(p + round);
      load_k();
      load_s(ks, 0);
      load_s(vs, 1);
      load_v();
      // (The last tile is a copy of the loop's body: a branch around the loads would make the
      // compiler wait for all of them.)
      for (; p + round < stop; p += round) {
        int n[2];
        place(n, p + round, stop, last, tail);
        fetch(p + 2 * round);
        tile(std::true_type{});
        count[0] = n[0];
        count[1] = n[1];
      }
      tile(std::false_type{});
    }

    l = across(l, [](float s, float t) { return s + t; });
    if (solo) {
      if (row < group) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < kDims; e += 4)
            write_out<D, kHalf>(a, b, head * group + row, (g * 4 + i) * (kDims / 4) + e / 4, m, l,
                                f32x4_t{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]});
      }
      continue;
    }
    // The waves' parts of the piece, joined in LDS.
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
    lds_barrier();
    float* part = a.parts + ((int64_t(head) * a.segments + segment) * 2 + (first > begin ? 1 : 0)) *
                                (int64_t(group) * (D + 4));
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
        write_out<D, kHalf>(a, b, head * group + r, c, top, sum, acc);
      } else {
        float* to = part + r * (D + 4);
        if (c == 0) *reinterpret_cast<float2*>(to) = make_float2(top, sum);
        *reinterpret_cast<f32x4_t*>(to + 4 + c * 4) = acc;
      }
    }
    lds_barrier();
  }

  // Requests without pages, or without any that are listed: zeros, and -inf.
  for (int i = segment; i < a.batch; i += whole_requests ? a.groups : a.segments) {
    if (min(indptr[i + 1] - base, total) > max(indptr[i] - base, 0)) continue;
    for (int j = threadIdx.x; j < group * D; j += kWaves * 64)
      a.out[i * a.out_stride + int64_t(head) * group * D + j] = 0;
    if (a.lse && int(threadIdx.x) < group)
      a.lse[int64_t(i) * a.hq + head * group + threadIdx.x] = -INFINITY;
  }
}

// Joins a request's pieces.  Workgroups (i, KV head, columns): request i, or in batches of more
// requests than there are borders between segments the request that border i + 1 cuts first; a
// column is four dims of a query row.  kShare neighbouring lanes take a column's pieces in turn and
// join theirs by DPP, without LDS: four registers that meet at each step, and no barrier.  What a
// launch of this takes (4 us) is its start and three loads that wait for each other.
template <int D, bool kHalf, int kShare>
__global__ __launch_bounds__(256) void quant_merge_kernel(QuantDecodeArgs a) {
  constexpr int kDeep = kShare >= 8 ? 1 : 2;   // pieces that a lane loads at a time
  const int head = blockIdx.x % a.hkv, i = blockIdx.x / a.hkv;
  const ScalarInts indptr = scalar_ints(a.indptr);
  const bool by_request = a.batch < a.segments;
  int b = by_request ? i : 0;
  const int base = indptr[0], total = pages_in_all(a, base, indptr[a.batch]);
  int first = indptr[b] - base, last = indptr[b + 1] - base;
  Search search;
  search.start(a.indptr, a.batch);
  if (share_of(a) != Share::cut) return;
  const int each = each_of(a.batch, total), all = total + each * a.batch;
  const int units = segment_units(a, all);
  const int64_t cut = int64_t(i + 1) * units;
  if (!by_request) {
    if (cut >= all) return;
    b = search.find(a.indptr, a.batch, base, int(cut), each, first, last);
  }
  if (first < 0) return;
  last = min(last, total) + each * (b + 1);
  first += each * (b + 1);
  if (last <= first || (!by_request && (first >= cut || first < cut - units))) return;
  const int s0 = uint32_t(first) / uint32_t(units);
  const int n = int(uint32_t(last - 1) / uint32_t(units)) - s0 + 1;
  if (n == 1) return;
  const int64_t step = int64_t(a.group) * (D + 4);
  const int64_t skip = first > int64_t(s0) * units ? step : 0;   // of the first piece's slot
  const int column = blockIdx.y * (256 / kShare) + threadIdx.x / kShare;
  const int r = min(column / (D / 4), a.group - 1), c = column % (D / 4);
  const float* parts = a.parts + (int64_t(head) * a.segments + s0) * 2 * step + r * (D + 4);
  float top = kLowest, sum = 0.f;
  f32x4_t acc = {};
  for (int s = threadIdx.x % kShare; s < n; s += kShare * kDeep) {
    float2 ml[kDeep];
    f32x4_t x[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int j = min(s + u * kShare, n - 1);
      const float* from = parts + j * 2 * step + (j == 0 ? skip : 0);
      ml[u] = *reinterpret_cast<const float2*>(from);
      x[u] = *reinterpret_cast<const f32x4_t*>(from + 4 + c * 4);
    }
    float most = top;
#pragma unroll
    for (int u = 0; u < kDeep; ++u) most = fmaxf(most, ml[u].x);
    float f = fast_exp2(top - most);
    sum *= f;
    acc *= f;
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
      if (s + u * kShare < n) {
        f = fast_exp2(ml[u].x - most);
        sum += ml[u].y * f;
        acc += x[u] * f;
      }
    top = most;
  }
  auto join = [](float v, auto f) {
    if constexpr (kShare >= 2) v = f(v, dpp<kDppQuadSwap1>(v));
    if constexpr (kShare >= 4) v = f(v, dpp<kDppQuadSwap2>(v));
    if constexpr (kShare >= 8) v = f(v, dpp<kDppRowHalfMirror>(v));
    if constexpr (kShare >= 16) v = f(v, dpp<kDppRowRor8>(v));
    if constexpr (kShare >= 64) v = across(v, f);
    return v;
  };
  const float mine = top;
  top = join(top, [](float x, float y) { return fmaxf(x, y); });
  const float f = fast_exp2(mine - top);
  sum = join(sum * f, [](float x, float y) { return x + y; });
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = join(acc[e] * f, [](float x, float y) { return x + y; });
  if (threadIdx.x % kShare == 0 && column < a.group * (D / 4))
    write_out<D, kHalf>(a, b, head * a.group + r, c, top, sum, acc);
}

// Segments per KV head.
int segments_of(int hkv, int head_dim) { return std::max(1, 256 * cut_for(head_dim) / hkv); }

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int64_t kvc_quantized_decode_workspace_bytes(int32_t batch, int32_t num_qo_heads,
                                                        int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
  return int64_t(segments_of(num_kv_heads, head_dim)) * 2 * num_qo_heads * (head_dim + 4) * 4;
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
  KVC_REQUIRE(num_indices <= INT32_MAX - 8 * 65536, KVC_ERR_INVALID_ARG, "too many indices");
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
  a.in_all = Divisor(uint32_t(a.segments));
  a.in_cus = Divisor(uint32_t(std::max(1, 256 / num_kv_heads)));
  // One request alone, whose segments are a piece each, is always faster with one per CU if that one
  // loads enough (8 KV heads of 128: 100000 tokens 37.9 -> 36.6 us, 10^6 307 -> 304; of 64, half the
  // bytes per token, 23.1 -> 25.5).
  a.even_from = batch == 1 && head_dim >= 128 ? INT32_MAX : 4 * kWaves;
  a.scale_log2 = sm_scale * kLog2e;
  a.parts = static_cast<float*>(workspace);
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_batch_stride;
  a.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  a.groups = std::max(a.segments, std::min(batch, 256 * per_simd(head_dim) / num_kv_heads));
  const unsigned grid = unsigned(a.groups) * unsigned(num_kv_heads);
  const unsigned lds = unsigned(kWaves * group * (head_dim + 4) * 4);
  // (So few pages are not cut, unless their requests are too many to look through.)
  const bool cut = a.segments > 1 &&
                   (num_indices > whole_pages(batch, num_kv_heads) || batch > kScan);

  auto launch = [&](auto d, auto c, auto half) {
    constexpr int D = decltype(d)::value, C = decltype(c)::value;
    constexpr bool H = decltype(half)::value;
    auto* kernel = &quant_decode_kernel<D, C, H>;
    if (lds > 65536)
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
    kernel<<<grid, kWaves * 64, lds, s>>>(a);
    if (cut) {
      const int joins = std::min(batch, a.segments - 1) * num_kv_heads;
      const unsigned columns = unsigned(group * (D / 4));
      // Lanes per column: as many as make up to 512 workgroups.  (3 requests of 2000 to 12000 tokens, 2 KV
      // heads of 256: 17.9 us with 4 lanes, 15.7 with 8, 14.6 with 16, 14.2 with 64; 64 of 512 to 4096, 8 of
      // 128: 57.6 with 2, 58.0 with 4, 59.3 with 8.)
      auto join = [&](auto lanes) {
        constexpr int S = decltype(lanes)::value;
        quant_merge_kernel<D, H, S>
            <<<dim3(unsigned(joins), (columns * S + 255) / 256), 256, 0, s>>>(a);
      };
      const int64_t room = 512 * 256 / (int64_t(joins) * columns);
      if (room >= 64)
        join(std::integral_constant<int, 64>{});
      else if (room >= 16)
        join(std::integral_constant<int, 16>{});
      else if (room >= 8)
        join(std::integral_constant<int, 8>{});
      else if (room >= 4)
        join(std::integral_constant<int, 4>{});
      else if (room >= 2)
        join(std::integral_constant<int, 2>{});
      else
        join(std::integral_constant<int, 1>{});
    }
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
