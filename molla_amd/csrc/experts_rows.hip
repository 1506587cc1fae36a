// experts_rows.hip -- experts_rows.h for Q4_K, Q6_K, Q4_0 and Q8_0 (the other kinds in
// experts_rows_more.hip, so that they compile in parallel).
#include "experts_rows.h"

namespace mi {

int launch_expert_rows_more(hipStream_t s, int kind, const ExpertRows& a);

bool one_row_fits(int32_t cols, int32_t share, int32_t pairs) { return share == pairs && cols <= kOneCols; }

int launch_expert_rows(hipStream_t s, int kind, const ExpertRows& a) {
  switch (kind) {
    case MI_Q4_K: return launch_rows_kind<MI_Q4_K>(s, a);
    case MI_Q6_K: return launch_rows_kind<MI_Q6_K>(s, a);
    case MI_Q4_0: return launch_rows_kind<MI_Q4_0>(s, a);
    case MI_Q8_0: return launch_rows_kind<MI_Q8_0>(s, a);
  }
  return launch_expert_rows_more(s, kind, a);
}

}  // namespace mi
