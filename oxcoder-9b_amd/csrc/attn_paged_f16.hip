// Attention over a paged cache of f16 values.
#include "attn_paged.h"

namespace kq {
template void launch_attn_part<KvF16>(const AttnArgs& a, hipStream_t s);
}
