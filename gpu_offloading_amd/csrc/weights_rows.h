// How a work unit of the attention weights' chunk form walks its query rows.
#pragma once

#include <hip/hip_runtime.h>

namespace kvc {

constexpr int kRows = 32;                          // query rows per block
constexpr int kStage = 2 * kRows;                  // rows in flight at a time

// Row i of a unit is token i / group, head i % group (tokens counted from the unit's
// first on).  A stage's rows are addressed by offsets from those of its first row's
// token; a row past the last token takes that token's place.
struct RowWalk {
  int group, step_tok, step_head;                  // a stage is so many tokens and heads on
  int last_tok;
  int tok, head;                                   // of the stage's first row

  __host__ __device__ __forceinline__ RowWalk(int group, int last_tok, int first_row)
      : group(group), step_tok(kStage / group), step_head(kStage % group), last_tok(last_tok),
        tok(first_row / group), head(first_row % group) {}
  // The last token, from the stage's first row's on.
  __host__ __device__ __forceinline__ int left() const { return last_tok - tok; }
  // On to the next stage, where there is one; returns the tokens between the bases.
  __host__ __device__ __forceinline__ int next() {
    int t = step_tok, h = head + step_head;
    if (h >= group) {
      h -= group;
      ++t;
    }
    if (tok + t > last_tok) return 0;
    tok += t;
    head = h;
    return t;
  }
  // Whether the rows' offsets may differ from those of the stage before: heads move, or
  // a row is past the last token.
  __host__ __device__ __forceinline__ bool offsets_change() const {
    return step_head != 0 || (left() + 1) * group < head + kStage;
  }
};

}  // namespace kvc
