// Attention of many rows: F16 queries over an E5M2 cache.
#include "kernels_attention_many.h"

namespace kvx {
namespace dev {

void run_attention_many_f16_e5m2(const AttentionArgs &a, bool vt, bool grouped, int64_t grid,
                                 hipStream_t s) {
  launch_many<KVX_DTYPE_F16, KVX_DTYPE_F8_E5M2>(a, vt, grouped, grid, s);
}

}  // namespace dev
}  // namespace kvx
