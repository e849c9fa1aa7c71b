// Attention over a paged cache of 8-bit codes.
#include "attn_paged.h"

namespace kq {
template void launch_attn_part<KvI8>(const AttnArgs& a, hipStream_t s);
}
