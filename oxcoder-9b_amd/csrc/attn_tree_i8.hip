// Attention of trees of drafted tokens over a paged cache of 8-bit codes.
#include "attn_tree.h"

namespace kq {
template void launch_attn_tree_part<KvI8>(const AttnArgs& a, hipStream_t s);
}
