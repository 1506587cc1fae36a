// experts_rows_more.hip -- experts_rows.h for Q4_1, Q5_0, Q5_1 and Q5_K.
#include "experts_rows.h"

namespace mi {

int launch_expert_rows_more(hipStream_t s, int kind, const ExpertRows& a) {
  switch (kind) {
    case MI_Q4_1: return launch_rows_kind<MI_Q4_1>(s, a);
    case MI_Q5_0: return launch_rows_kind<MI_Q5_0>(s, a);
    case MI_Q5_1: return launch_rows_kind<MI_Q5_1>(s, a);
    case MI_Q5_K: return launch_rows_kind<MI_Q5_K>(s, a);
  }
  return fail(MI_ERR_KIND, "experts: ggml type %d has no device kernel", kind);
}

}  // namespace mi
