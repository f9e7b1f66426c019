// Attention of few rows: BF16 queries over a BF16 cache.
#include "kernels_attention_few.h"

namespace kvx {
namespace dev {

void run_attention_few_bf16(const AttentionPart &p, bool vt, bool grouped, hipStream_t s) {
  launch_few<KVX_DTYPE_BF16, KVX_DTYPE_BF16>(p, vt, grouped, s);
}

}  // namespace dev
}  // namespace kvx
