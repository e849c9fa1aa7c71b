// Attention over a paged cache of bf16 values.
#include "attn_paged.h"

namespace kq {
template void launch_attn_part<KvBf16, false>(const AttnArgs& a, hipStream_t s);
}
