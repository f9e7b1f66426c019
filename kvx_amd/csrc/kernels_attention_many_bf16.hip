// Attention of many rows: BF16 queries over a BF16 cache.
#include "kernels_attention_many.h"

namespace kvx {
namespace dev {

void run_attention_many_bf16(const AttentionArgs &a, bool vt, bool grouped, int64_t grid,
                             hipStream_t s) {
  launch_many<KVX_DTYPE_BF16, KVX_DTYPE_BF16>(a, vt, grouped, grid, s);
}

}  // namespace dev
}  // namespace kvx
