// Attention of trees of drafted tokens over a paged cache of f16 values.
#include "attn_tree.h"

namespace kq {
template void launch_attn_tree_part<KvF16>(const AttnArgs& a, hipStream_t s);
}
