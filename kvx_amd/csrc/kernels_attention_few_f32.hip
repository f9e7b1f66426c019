// Attention of few rows: F32 queries over an F32 cache.
#include "kernels_attention_few.h"

namespace kvx {
namespace dev {

void run_attention_few_f32(const AttentionPart &p, bool vt, bool grouped, hipStream_t s) {
  launch_few<KVX_DTYPE_F32, KVX_DTYPE_F32>(p, vt, grouped, s);
}

}  // namespace dev
}  // namespace kvx
