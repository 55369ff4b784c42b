// The float16 kernels of paged_attention.hpp.
#include "paged_attention.hpp"

namespace cbk {

int launch_paged_attention_f16(const PagedAttnArgs& a, int64_t head_dim, hipStream_t s) {
  return launch_type<CBK_DTYPE_F16>(a, head_dim, s);
}

}  // namespace cbk
