// Attention of few rows: F16 queries over an E5M2 cache.
#include "kernels_attention_few.h"

namespace kvx {
namespace dev {

void run_attention_few_f16_e5m2(const AttentionPart &p, bool vt, bool grouped, hipStream_t s) {
  launch_few<KVX_DTYPE_F16, KVX_DTYPE_F8_E5M2>(p, vt, grouped, s);
}

}  // namespace dev
}  // namespace kvx
