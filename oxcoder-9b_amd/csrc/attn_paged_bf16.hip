// Attention over a paged cache of bf16 values.
#include "attn_paged.h"

namespace kq {
template void launch_attn_part<KvBf16>(const AttnArgs& a, hipStream_t s);
}
