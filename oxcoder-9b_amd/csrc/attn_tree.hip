// Attention of trees of drafted tokens over a paged key-value cache (include/kq.h: kq_attn_tree): how the positions are
// split, and the join of the parts that attn_tree.h's kernels leave.
#include "attn_tree.h"

namespace kq {

// ROWS rows a workgroup, 256 / ROWS threads each: lanes of 4 values, in groups that take every so many parts.
template <int ROWS>
__global__ void __launch_bounds__(256) k_attn_tree_join(AttnArgs a, int lanes) {
    __shared__ f32x4 so[256];
    __shared__ float sl[256];
    const int tid = threadIdx.x, per = 256 / ROWS, groups = per / lanes, at = tid % per, group = at / lanes, d = 4 * (at % lanes);
    const int D = a.kv.dim, G = a.group, H = a.q_heads;
    const int64_t i = (int64_t)blockIdx.x * ROWS + tid / per, rows = (int64_t)a.table.seqs * a.T * H;
    const int64_t bt = min(i, rows - 1) / H;
    const int h = (int)(min(i, rows - 1) % H), b = (int)(bt / a.T), t = (int)(bt % a.T);
    const int len = tree_length(a, a.lens[b]), n = (len + a.split - 1) / a.split;
    const int64_t row = (((int64_t)b * a.kv.heads + h / G) * a.T * G + t * G + h % G) * a.parts;
    float top = -INFINITY;
    for (int c = 0; c < n; c++) top = fmaxf(top, a.pml[row + c].m);
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f;
    if (group < groups && d < D)
        for (int c = group; c < n; c += groups) {
            const AttnMl ml = a.pml[row + c];
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.po + (row + c) * D + d);
            const float k = ml.l != 0.0f ? __builtin_amdgcn_exp2f(ml.m - top) : 0.0f;   // 0: the row saw nothing (a NaN counts)
            if (ml.l != 0.0f) sum += x * k;
            total += ml.l * k;
        }
    if (groups > 1) {
        so[tid] = sum, sl[tid] = total;
        __syncthreads();
        if (group == 0)
            for (int w = 1; w < groups; w++) sum += so[tid + w * lanes], total += sl[tid + w * lanes];
    }
    if (group == 0 && d < D && i < rows)
        *reinterpret_cast<f32x4_a4*>(a.out + bt * a.ldo + (int64_t)h * D + d) = total == 0.0f ? f32x4{0, 0, 0, 0} : sum / total;
}

struct TreeSplit {
    int tiles, split, parts;   // 16 rows each that a wave takes; positions of a part; parts
};
// How a call's rows and positions are shared out.
static TreeSplit split_of(int seqs, int heads, int group, int dim, int T, int max_len) {
    TreeSplit s;
    const int R = T * group;
    s.tiles = R <= 64 || dim > 128 ? 1 : 2;
    const int64_t columns = (int64_t)seqs * heads * ((R + 64 * s.tiles - 1) / (64 * s.tiles));
    const int64_t want = (2048 + columns - 1) / columns;
    int64_t split = (max_len + want - 1) / want;
    if (split < 64) split = 64;
    if (split < (max_len + 65534) / 65535) split = (max_len + 65534) / 65535;
    split = (split + 31) / 32 * 32;
    s.split = (int)split;
    s.parts = (int)((max_len + split - 1) / split);
    return s;
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t attn_tree_bytes(int seqs, int heads, int group, int dim, int T, int max_len) {
    const TreeSplit s = split_of(seqs, heads, group, dim, T, max_len);
    const size_t parts = (size_t)seqs * T * heads * group * s.parts;
    return s.parts == 1 ? 256 : up256(parts * dim * 4) + up256(parts * sizeof(AttnMl));
}

// What trees of up to T nodes need, whatever the key-value heads.
size_t attn_tree_workspace(int seqs, int q_heads, int dim, int T, int max_len) {
    size_t most = 256;
    for (int heads = 1; heads <= q_heads; heads++)
        for (int t = 1; t <= T && q_heads % heads == 0; t++) {
            const size_t n = attn_tree_bytes(seqs, heads, q_heads / heads, dim, t, max_len);
            most = n > most ? n : most;
        }
    return most;
}

void launch_attn_tree(const AttnArgs& args, hipStream_t s) {
    AttnArgs a = args;
    a.scale *= 1.44269504088896341f;                           // scores in powers of 2
    a.group = a.q_heads / a.kv.heads;
    a.page_shift = __builtin_ctz((unsigned)a.kv.page_size);
    const TreeSplit w = split_of(a.table.seqs, a.kv.heads, a.group, a.kv.dim, a.T, a.bound);
    a.tiles = w.tiles, a.split = w.split, a.parts = w.parts;
    a.joined = a.parts > 1;
    const size_t parts = (size_t)a.table.seqs * a.T * a.q_heads * a.parts;
    a.po = reinterpret_cast<float*>(a.ws);
    a.pml = reinterpret_cast<AttnMl*>(a.ws + up256(parts * a.kv.dim * 4));
    if (a.kv.type == KQ_KV_F16) launch_attn_tree_part<KvF16>(a, s);
    else if (a.kv.type == KQ_KV_BF16) launch_attn_tree_part<KvBf16>(a, s);
    else launch_attn_tree_part<KvI8>(a, s);
    if (!a.joined) return;
    const int64_t rows = (int64_t)a.table.seqs * a.T * a.q_heads;
    const int lanes = a.kv.dim <= 64 ? 16 : a.kv.dim <= 128 ? 32 : 64;
    if (a.parts <= 16 && lanes <= 32) hipLaunchKernelGGL(k_attn_tree_join<8>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a, lanes);
    else if (a.parts <= 16) hipLaunchKernelGGL(k_attn_tree_join<4>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, lanes);
    else hipLaunchKernelGGL(k_attn_tree_join<1>, dim3((unsigned)rows), dim3(256), 0, s, a, lanes);
}

}  // namespace kq
