// Attention of trees of drafted tokens over a paged cache of bf16 values.
#include "attn_tree.h"

namespace kq {
template void launch_attn_tree_part<KvBf16>(const AttnArgs& a, hipStream_t s);
}
