// Attention of single tokens over a paged cache, f16.
#include "paged_attention_kernel.h"

namespace fr {
template int paged_attention_run<f16_t>(const fr_paged_args&, int64_t, int, hipStream_t);
}  // namespace fr
