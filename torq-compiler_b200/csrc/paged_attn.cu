// Which kernel takes which rows of attn_paged.
#include "kernels.h"

namespace tb200 {

cudaError_t launch_attn_paged(AttnPagedArgs a, cudaStream_t stream) {
  a.few_rows = 0;
  return launch_attn_paged_tile(a, stream);
}

}  // namespace tb200
