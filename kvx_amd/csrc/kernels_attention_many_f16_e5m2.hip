// Attention of many rows: F16 queries over an E5M2 cache.
#include "kernels_attention_many.h"

namespace kvx {
namespace dev {

void run_attention_many_f16_e5m2(const AttentionPart &p, const AttentionPart *few, bool vt,
                                 bool grouped, hipStream_t s) {
  launch_many<KVX_DTYPE_F16, KVX_DTYPE_F8_E5M2>(p, few, vt, grouped, s);
}

}  // namespace dev
}  // namespace kvx
