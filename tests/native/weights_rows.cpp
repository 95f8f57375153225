// Replays, on the CPU, where the attention weights' chunk kernel reads its query rows:
// every unit of kvc_weights_plan walked as the kernel walks it (csrc/weights_rows.h).
// Offsets are computed when the walk says that they change and else kept, so a kept one
// that no longer fits shows.  Every row must read a token of its unit, and a row of the
// unit's blocks its own token and head.  Prints "ok <units>", or the first violation.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "kvc.h"
#include "weights_rows.h"

using kvc::kRows;
using kvc::kStage;

int main() {
  const int lengths[][3] = {{1, 1, 1}, {2, 3, 1}, {5, 129, 33}, {129, 777, 2}, {1000, 64, 65}};
  long units = 0, cut_units = 0, large_cut = 0;
  for (int group = 1; group <= 128; ++group)
    for (int hkv = 1; hkv <= 2; ++hkv)
      for (const int d : {64, 128, 256})
        for (const int causal : {0, 1})
          for (const auto& q : lengths) {
            std::vector<int32_t> qo = {0}, kv = {0}, lpl;
            for (int b = 0; b < 3; ++b) {
              const int len = q[b] + 7 * b;
              qo.push_back(qo.back() + q[b]);
              kv.push_back(kv.back() + (len + 15) / 16);
              lpl.push_back((len - 1) % 16 + 1);
            }
            kvc_weights_schedule s;
            std::vector<int32_t> img(1 << 18);
            if (kvc_weights_plan(qo.data(), kv.data(), lpl.data(), nullptr, 3, hkv * group, hkv, d,
                                 16, causal, &s, img.data(), int64_t(img.size()))) {
              std::printf("plan: %s\n", kvc_last_error());
              return 1;
            }
            for (int u = 0; u < s.num_units; ++u) {
              const int32_t* r = img.data() + 12 * u;
              const int key0 = r[1], q_len = r[2], kv_len = r[3], first = r[8], blocks = r[9];
              const int before = key0 - (kv_len - q_len);
              const int tok0 = causal && before > 0 ? before : 0;
              const int stages = (blocks + 1) / 2, last = q_len - 1 - tok0;
              ++units;
              if (r[10] >= 0) ++cut_units, large_cut += group > 32;
              if (stages == 0) continue;
              kvc::RowWalk at(group, last, first * kRows);
              int tok[kStage], head[kStage], base = at.tok;
              auto offsets = [&] {
                for (int i = 0; i < kStage; ++i) {
                  tok[i] = std::min((at.head + i) / group, at.left());
                  head[i] = (at.head + i) % group;
                }
              };
              offsets();
              // (the kernel loads one stage more than it computes)
              for (int st = 0; st <= stages; ++st) {
                for (int i = 0; i < kStage; ++i) {
                  const int row = first * kRows + st * kStage + i;
                  const bool mine = st * kStage + i < blocks * kRows && row / group <= last;
                  if (base + tok[i] < 0 || base + tok[i] > last || head[i] >= group ||
                      (mine && (base + tok[i] != row / group || head[i] != row % group))) {
                    std::printf("group %d, %d KV heads, head_dim %d, causal %d, queries %d %d %d, "
                                "unit %d (blocks %d..%d), stage %d, row %d: token %d of %d\n",
                                group, hkv, d, causal, q[0], q[1], q[2], u, first, first + blocks,
                                st, i, base + tok[i], last + 1);
                    return 1;
                  }
                }
                base += at.next();
                if (at.offsets_change()) offsets();
              }
            }
          }
  if (cut_units == 0 || large_cut == 0) {
    std::printf("no unit was cut\n");
    return 1;
  }
  std::printf("ok %ld\n", units);
  return 0;
}
