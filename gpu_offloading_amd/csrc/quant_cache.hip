// Writing the quantised cache (quant.h) and reading it back.
//
// Layout: codes [blocks][heads][16][D] for K and for V, so that a block's tile of one head
// is contiguous (2 KB at D = 128), scales fp32 [blocks][heads][2][16], K's and V's of a tile in
// one 128-byte line: the decode reads both with the tile.
//
// Both kernels move bytes (three per value, and the scales) and are bound by them.  The unit is a
// row, one token's D values of one head: D / 8 lanes with 8 values each, 16 bytes of the
// model's type and 8 of codes, so that both sides are whole lines.  Rows are dealt tile by
// tile (16 tokens of a head, K and V in turn): 16 neighbouring tokens' codes are one
// contiguous piece of the cache, and their scales one line that a workgroup completes.
// Rows of the model's type move with the non-temporal hint (32768 tokens written 40.4 -> 38.8 us,
// read back 42.4 -> 38.9), codes without: a chunk's are read back in the same step, and 16384 tokens
// written and read back take 35.6 us in place of 40.0 by stores that stay in the caches.  The write
// alone takes longer by them, 42.0 us for 38.9 at 32768 tokens: a new prompt, whose codes no one reads in
// its step, pays that.  (A decode step's write is too small to show either; write and attention were not
// timed together both ways.)  Histories that fit the 256 MB cache in front of the memory are read from
// there (8 x 4096 tokens 38.6 -> 30.8 us; 41.5 for 40.5 where they do not).  A large device copy reaches
// 5.1 TB/s; these 4.9 and 4.9, from memory, and 4.7 and 6.6 from the cache.
#include "quant.h"

#include <algorithm>
#include <type_traits>

namespace kvc {
namespace {

constexpr int kThreads = 256;

// Largest of a row's packed 16-bit absolute bit patterns over its kLanes lanes.
template <int kLanes>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  auto up = [&](uint32_t o) {
    v = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, v),
                                                               __builtin_bit_cast(u16x2_t, o)));
  };
  auto dpp_of = [&](auto c) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), decltype(c)::value, 0xF, 0xF, true));
  };
  up(dpp_of(std::integral_constant<int, kDppQuadSwap1>{}));
  up(dpp_of(std::integral_constant<int, kDppQuadSwap2>{}));
  up(dpp_of(std::integral_constant<int, kDppRowHalfMirror>{}));
  if constexpr (kLanes >= 16) up(dpp_of(std::integral_constant<int, kDppRowRor8>{}));
  if constexpr (kLanes >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = s[0];
    up(s[1]);
  }
  return max(v & 0xffffu, v >> 16);
}

struct WriteArgs {
  const uint16_t* src[2];   // key, value
  uint8_t* cache[2];
  float* scales;
  const int64_t* slots;
  uint32_t num_tokens;
  int64_t src_stride[2];    // elements between tokens
  int64_t block_stride;     // codes between blocks
  int64_t scales_stride;    // floats between blocks
  int64_t num_slots;
  int32_t heads;
  int32_t* oob_count;
};

// kVec: the rows are 16-byte aligned; otherwise their values are loaded one by one.
template <int D, int kCode, bool kHalf, bool kVec, int kUnroll>
__global__ __launch_bounds__(kThreads) void quant_write_kernel(WriteArgs a) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  // (the host keeps the rows of a call below 2^31)
  const uint32_t row0 = blockIdx.x * uint32_t(kRows * kUnroll) + threadIdx.x / kLanes;
  uint4 x[kUnroll];
  int64_t slot[kUnroll];
  int head[kUnroll], kv[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t row = row0 + u * kRows, tile = row / kQuantPage;
    const uint32_t group = tile / uint32_t(2 * a.heads), pair = tile - group * uint32_t(2 * a.heads);
    const uint32_t token = group * kQuantPage + row % kQuantPage;
    kv[u] = pair & 1;
    head[u] = pair >> 1;
    slot[u] = -1;
    x[u] = make_uint4(0, 0, 0, 0);
    if (token >= a.num_tokens) continue;
    slot[u] = a.slots[token];
    const uint16_t* p = (kv[u] ? a.src[1] : a.src[0]) +
                        token * (kv[u] ? a.src_stride[1] : a.src_stride[0]) +
                        head[u] * D + lane * 8;
    if constexpr (kVec) {
      x[u] = load_stream(p);
    } else {
      x[u] = make_uint4(p[0] | uint32_t(p[1]) << 16, p[2] | uint32_t(p[3]) << 16,
                        p[4] | uint32_t(p[5]) << 16, p[6] | uint32_t(p[7]) << 16);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most = __builtin_bit_cast(
          uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, most),
                                              __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu)));
    most = row_max<kLanes>(most);   // (all lanes, whatever their slots)
    const RowScale s = row_scale<kCode, kHalf>(__float_as_uint(unpack_lo<kHalf>(most)));
    if (slot[u] < 0) continue;
    if (slot[u] >= a.num_slots) {
      if (a.oob_count && lane == 0 && head[u] == 0 && kv[u] == 0) atomicAdd(a.oob_count, 1);
      continue;
    }
    const int64_t block = slot[u] >> 4;
    const int place = int(slot[u]) & 15;
    uint2 c;
    c.x = encode4<kCode>(unpack_lo<kHalf>(w[0]), unpack_hi<kHalf>(w[0]), unpack_lo<kHalf>(w[1]),
                         unpack_hi<kHalf>(w[1]), s);
    c.y = encode4<kCode>(unpack_lo<kHalf>(w[2]), unpack_hi<kHalf>(w[2]), unpack_lo<kHalf>(w[3]),
                         unpack_hi<kHalf>(w[3]), s);
    uint8_t* to = (kv[u] ? a.cache[1] : a.cache[0]) + block * a.block_stride +
                  (head[u] * kQuantPage + place) * D + lane * 8;
    *reinterpret_cast<uint2*>(to) = c;
    if (lane == 0)
      a.scales[block * a.scales_stride + (head[u] * 2 + kv[u]) * kQuantPage + place] = s.scale;
  }
}

struct ReadArgs {
  const uint8_t* cache[2];
  const float* scales;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t bt_width;
  const int32_t* cu_seq_lens;
  const int32_t* seq_starts;   // may be null
  int64_t block_stride, scales_stride, num_blocks;
  uint16_t* out[2];
  int64_t out_stride;          // elements between output rows
  int64_t out_rows;
  int32_t max_seq_len;
  int32_t heads;
  int32_t* oob_count;
};

// Workgroup (page of a sequence, sequence, batch of rows): kRows * kUnroll rows of the page.
template <int D, int kCode, bool kHalf, bool kVec, int kUnroll>
__global__ __launch_bounds__(kThreads) void quant_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int b = blockIdx.y;
  const int64_t first = a.cu_seq_lens[b];
  const int64_t len = min(a.cu_seq_lens[b + 1] - first, int64_t(a.max_seq_len));
  const int64_t start = a.seq_starts ? a.seq_starts[b] : 0;
  // Pages are counted from the one that holds token `start` (rounded down, also below 0).
  const int64_t page = (start >> 4) + blockIdx.x;
  if (len <= 0 || page * kQuantPage >= start + len) return;
  const int64_t id = page >= 0 && page < a.bt_width ? a.block_table[b * a.bt_stride + page] : -1;
  const bool held = id >= 0 && id < a.num_blocks;
  const int row0 = blockIdx.z * (kRows * kUnroll) + threadIdx.x / kLanes;
  uint2 c[kUnroll];
  float scale[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int row = row0 + u * kRows, pair = row / kQuantPage, place = row % kQuantPage;
    c[u] = make_uint2(0, 0);
    scale[u] = 0.f;
    const int64_t t = page * kQuantPage + place - start;
    if (!held || pair >= 2 * a.heads || t < 0 || t >= len) continue;
    const int kv = pair & 1, head = pair >> 1;
    const uint8_t* p = (kv ? a.cache[1] : a.cache[0]) + id * a.block_stride +
                       (head * kQuantPage + place) * D + lane * 8;
    c[u] = *reinterpret_cast<const uint2*>(p);
    scale[u] = a.scales[id * a.scales_stride + (head * 2 + kv) * kQuantPage + place];
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int row = row0 + u * kRows, pair = row / kQuantPage, place = row % kQuantPage;
    const int64_t t = page * kQuantPage + place - start;
    if (pair >= 2 * a.heads || t < 0 || t >= len) continue;
    const bool inside = first + t >= 0 && first + t < a.out_rows;
    if (a.oob_count && lane == 0 && pair == 0 && !(inside && held)) atomicAdd(a.oob_count, 1);
    if (!inside) continue;
    const uint32_t w[2] = {c[u].x, c[u].y};
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[2 * i] = pack2<kHalf>(decode1<kCode, 0>(w[i]) * scale[u],
                              decode1<kCode, 1>(w[i]) * scale[u]);
      v[2 * i + 1] = pack2<kHalf>(decode1<kCode, 2>(w[i]) * scale[u],
                                  decode1<kCode, 3>(w[i]) * scale[u]);
    }
    uint16_t* to = ((pair & 1) ? a.out[1] : a.out[0]) + (first + t) * a.out_stride +
                   (pair >> 1) * D + lane * 8;
    if constexpr (kVec) {
      store_stream(to, make_uint4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        to[2 * i] = uint16_t(v[i]);
        to[2 * i + 1] = uint16_t(v[i] >> 16);
      }
    }
  }
}

// Calls f with the compile-time (head_dim, code, type) of a call.
template <typename F>
bool with_types(int32_t head_dim, int32_t code, int32_t dtype, F&& f) {
  auto by_type = [&](auto d, auto c) {
    if (dtype == KVC_DTYPE_FP16)
      f(d, c, std::true_type{});
    else
      f(d, c, std::false_type{});
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
  else if (head_dim == 256)
    by_code(std::integral_constant<int, 256>{});
  else
    return false;
  return true;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

#define KVC_REQUIRE_QUANT(key_cache, value_cache, scales, code, dtype)                       \
  KVC_REQUIRE(code == KVC_CODE_E4M3 || code == KVC_CODE_INT8, KVC_ERR_UNSUPPORTED,            \
              "code must be KVC_CODE_E4M3 or KVC_CODE_INT8");                                 \
  KVC_REQUIRE(dtype == KVC_DTYPE_FP16 || dtype == KVC_DTYPE_BF16, KVC_ERR_UNSUPPORTED,        \
              "dtype must be KVC_DTYPE_FP16 or KVC_DTYPE_BF16");                              \
  KVC_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535 && num_blocks > 0,                    \
              KVC_ERR_INVALID_ARG, "non-positive shape or too many heads");                   \
  KVC_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, KVC_ERR_UNSUPPORTED,      \
              "head_dim must be 64, 128 or 256");                                             \
  KVC_REQUIRE(block_size == kQuantPage, KVC_ERR_UNSUPPORTED, "block_size must be 16");        \
  KVC_REQUIRE(cache_block_stride >= int64_t(num_kv_heads) * kQuantPage * head_dim &&          \
                  scales_block_stride >= int64_t(num_kv_heads) * 2 * kQuantPage,              \
              KVC_ERR_INVALID_ARG, "a block stride is smaller than a block");                 \
  KVC_REQUIRE(aligned(key_cache, 16) && aligned(value_cache, 16) && aligned(scales, 16) &&    \
                  cache_block_stride % 16 == 0 && scales_block_stride % 4 == 0,               \
              KVC_ERR_ALIGNMENT, "the caches, the scales and their block strides must be "    \
                                 "multiples of 16 bytes")

extern "C" int kvc_reshape_and_cache_quantized(
    const void* key, const void* value, void* key_cache, void* value_cache, float* scales,
    const int64_t* slot_mapping, int64_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, int64_t num_blocks, int32_t dtype, int32_t code,
    int64_t key_token_stride, int64_t value_token_stride, int64_t cache_block_stride,
    int64_t scales_block_stride, int32_t* oob_count, void* stream) {
  KVC_REQUIRE(num_tokens >= 0, KVC_ERR_INVALID_ARG, "num_tokens < 0");
  if (num_tokens == 0) return ok();
  KVC_REQUIRE(key && value && key_cache && value_cache && scales && slot_mapping,
              KVC_ERR_INVALID_ARG, "null pointer");
  KVC_REQUIRE_QUANT(key_cache, value_cache, scales, code, dtype);
  const int64_t row = int64_t(num_kv_heads) * head_dim;
  KVC_REQUIRE(key_token_stride >= row && value_token_stride >= row, KVC_ERR_INVALID_ARG,
              "source token stride smaller than a row");
  KVC_REQUIRE(aligned(key, 2) && aligned(value, 2), KVC_ERR_ALIGNMENT,
              "key and value must be aligned to their type");
  const int64_t rows = (num_tokens + kQuantPage - 1) / kQuantPage * kQuantPage * 2 * num_kv_heads;
  // (A launch has less than 2^32 threads; a workgroup moves 2048 values.)
  KVC_REQUIRE(num_tokens < (int64_t(1) << 31) && rows * head_dim <= (int64_t(1) << 35) - 2048,
              KVC_ERR_INVALID_ARG, "too many tokens in one call; split the batch");

  WriteArgs a;
  a.src[0] = static_cast<const uint16_t*>(key);
  a.src[1] = static_cast<const uint16_t*>(value);
  a.cache[0] = static_cast<uint8_t*>(key_cache);
  a.cache[1] = static_cast<uint8_t*>(value_cache);
  a.scales = scales;
  a.slots = slot_mapping;
  a.num_tokens = uint32_t(num_tokens);
  a.src_stride[0] = key_token_stride;
  a.src_stride[1] = value_token_stride;
  a.block_stride = cache_block_stride;
  a.scales_stride = scales_block_stride;
  a.num_slots = num_blocks * kQuantPage;
  a.heads = num_kv_heads;
  a.oob_count = oob_count;
  const bool vec = aligned(key, 16) && aligned(value, 16) && key_token_stride % 8 == 0 &&
                   value_token_stride % 8 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(head_dim, code, dtype, [&](auto d, auto c, auto half) {
    constexpr int D = decltype(d)::value, C = decltype(c)::value;
    constexpr bool H = decltype(half)::value;
    constexpr int kRows = kThreads / (D / 8);
    const unsigned groups = unsigned((rows + kRows - 1) / kRows);
    // Rows per thread: few tokens want many workgroups (64 of 8 x 128: 2.2 us with 1, 3.4 with 4),
    // many want loads in flight (10000 of 4 x 256: 13.2 us with 4, 14.0 with 2, 15.3 with 1; 4096
    // of 8 x 128: 6.7 with 2, 6.8 with 4, 7.3 with 1).
    if (!vec)
      quant_write_kernel<D, C, H, false, 1><<<groups, kThreads, 0, s>>>(a);
    else if (groups <= 1024)
      quant_write_kernel<D, C, H, true, 1><<<groups, kThreads, 0, s>>>(a);
    else if (groups < 8192)
      quant_write_kernel<D, C, H, true, 2><<<(groups + 1) / 2, kThreads, 0, s>>>(a);
    else
      quant_write_kernel<D, C, H, true, 4><<<(groups + 3) / 4, kThreads, 0, s>>>(a);
  });
  KVC_LAUNCH_CHECK();
  return ok();
}

extern "C" int kvc_gather_quantized_kv(
    const void* key_cache, const void* value_cache, const float* scales,
    const int32_t* block_table, int64_t block_table_row_stride, int32_t block_table_width,
    const int32_t* cu_seq_lens, const int32_t* seq_starts, int32_t batch, int32_t max_seq_len,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int64_t num_blocks,
    int32_t dtype, int32_t code, int64_t cache_block_stride, int64_t scales_block_stride,
    void* out_key, void* out_value, int64_t out_token_stride, int64_t out_rows,
    int32_t* oob_count, void* stream) {
  KVC_REQUIRE(batch >= 0 && max_seq_len >= 0 && out_rows >= 0, KVC_ERR_INVALID_ARG,
              "negative batch, max_seq_len or out_rows");
  if (batch == 0 || max_seq_len == 0) return ok();
  KVC_REQUIRE(key_cache && value_cache && scales && block_table && cu_seq_lens && out_key &&
                  out_value,
              KVC_ERR_INVALID_ARG, "null pointer");
  KVC_REQUIRE(batch <= 65535, KVC_ERR_INVALID_ARG, "batch > 65535");
  KVC_REQUIRE(block_table_width > 0, KVC_ERR_INVALID_ARG, "non-positive block table width");
  KVC_REQUIRE_QUANT(key_cache, value_cache, scales, code, dtype);
  KVC_REQUIRE(out_token_stride >= int64_t(num_kv_heads) * head_dim, KVC_ERR_INVALID_ARG,
              "output token stride smaller than a row");
  KVC_REQUIRE(aligned(out_key, 2) && aligned(out_value, 2), KVC_ERR_ALIGNMENT,
              "the outputs must be aligned to their type");

  ReadArgs a;
  a.cache[0] = static_cast<const uint8_t*>(key_cache);
  a.cache[1] = static_cast<const uint8_t*>(value_cache);
  a.scales = scales;
  a.block_table = block_table;
  a.bt_stride = block_table_row_stride;
  a.bt_width = block_table_width;
  a.cu_seq_lens = cu_seq_lens;
  a.seq_starts = seq_starts;
  a.block_stride = cache_block_stride;
  a.scales_stride = scales_block_stride;
  a.num_blocks = num_blocks;
  a.out[0] = static_cast<uint16_t*>(out_key);
  a.out[1] = static_cast<uint16_t*>(out_value);
  a.out_stride = out_token_stride;
  a.out_rows = out_rows;
  a.max_seq_len = max_seq_len;
  a.heads = num_kv_heads;
  a.oob_count = oob_count;
  const bool vec = aligned(out_key, 16) && aligned(out_value, 16) && out_token_stride % 8 == 0;
  // One page more than max_seq_len fills where a range may begin inside one.
  const unsigned pages = unsigned(cdiv(max_seq_len, kQuantPage)) + (seq_starts ? 1u : 0u);
  const int64_t rows = int64_t(num_kv_heads) * 2 * kQuantPage;
  KVC_REQUIRE(pages < (1u << 24) && rows * head_dim <= 65535 * 2048, KVC_ERR_INVALID_ARG,
              "max_seq_len or num_kv_heads too large for one call");
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_types(head_dim, code, dtype, [&](auto d, auto c, auto half) {
    constexpr int D = decltype(d)::value, C = decltype(c)::value;
    constexpr bool H = decltype(half)::value;
    constexpr int kRows = kThreads / (D / 8);
    const unsigned batches = unsigned((rows + kRows - 1) / kRows);
    // Rows per thread, as for the write (64 x 1 token of 8 x 128: 2.8 us with 1, 3.4 with 4; 20 ragged
    // sequences of up to 3000: 42.6 with 4, 43.9 with 8, 44.8 with 2, 48.9 with 1).
    if (!vec)
      quant_read_kernel<D, C, H, false, 1><<<dim3(pages, batch, batches), kThreads, 0, s>>>(a);
    else if (int64_t(pages) * batch * batches <= 1024)
      quant_read_kernel<D, C, H, true, 1><<<dim3(pages, batch, batches), kThreads, 0, s>>>(a);
    else
      quant_read_kernel<D, C, H, true, 4><<<dim3(pages, batch, (batches + 3) / 4), kThreads, 0, s>>>(a);
  });
  KVC_LAUNCH_CHECK();
  return ok();
}
