// Attention of trees of drafted tokens over a paged key-value cache (include/kq.h: kq_attn_tree): how the positions are
// split, and the join of the parts that attn_tree.h's kernels leave.
#include <math.h>

#include "kv_device.h"

namespace kq {

// ROWS rows a workgroup, 256 / ROWS threads each: lanes of 4 values, in groups that take every so many parts.  The parts'
// largest scores and sums are looked at by all of a row's threads, and their weights left in LDS.  Bound by the parts' bytes and the
// chain of loads: 4.3 us for 256 rows of 20 parts, 9.4 for 2048 of 32 (34 MB).
constexpr int TJ_MOST = 2048;                // parts of a row at most
template <int ROWS>
__global__ void __launch_bounds__(256) k_attn_tree_join(AttnArgs a, int lanes) {
    extern __shared__ float weight[];                          // [row][part], then the groups' sums
    __shared__ float stat[ROWS];
    const int per = 256 / ROWS, mine = threadIdx.x / per, at = threadIdx.x % per, groups = per / lanes, group = at / lanes;
    const int d = 4 * (at % lanes), D = a.kv.dim, G = a.group, H = a.q_heads;
    const int64_t rows = (int64_t)a.table.seqs * a.T * H, i = min((int64_t)blockIdx.x * ROWS + mine, rows - 1), bt = i / H;
    const int h = (int)(i % H), b = (int)(bt / a.T), t = (int)(bt % a.T);
    const int len = tree_length(a, a.lens[b]), n = (len + a.split - 1) / a.split;
    const int64_t row = (((int64_t)b * a.kv.heads + h / G) * a.T * G + t * G + h % G) * a.parts;
    float* const w = weight + mine * a.parts;
    // the first wave of a row's threads (or the part of one that they are)
    if (at < 64) {
        const int step = min(per, 64);
        float top = -INFINITY, total = 0.0f;
        for (int c = at; c < n; c += step) top = fmaxf(top, a.pml[row + c].m);
        for (int x = step >> 1; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        for (int c = at; c < n; c += step) {
            const AttnMl ml = a.pml[row + c];
            const float k = ml.l != 0.0f ? __builtin_amdgcn_exp2f(ml.m - top) : 0.0f;   // 0: the row saw nothing (a NaN counts)
            w[c] = k;
            total += ml.l * k;
        }
        for (int x = step >> 1; x; x >>= 1) total += __shfl_xor(total, x, 64);
        if (at == 0) stat[mine] = total;
    }
    __syncthreads();
    f32x4 sum = {0, 0, 0, 0};
    if (d < D) {
        const float* po = a.po + row * D + d;
#pragma unroll 4
        for (int c = group; c < n; c += groups) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(po + (int64_t)c * D);
            const float k = w[c];
            // an infinity or NaN that the row saw counts however small the part's weight
#pragma unroll
            for (int i = 0; i < 4; i++) sum[i] += k != 0.0f ? x[i] * k : fabsf(x[i]) < INFINITY ? 0.0f : x[i];
        }
    }
    if (groups > 1) {
        f32x4* so = reinterpret_cast<f32x4*>(weight + (ROWS * a.parts + 3) / 4 * 4);
        so[threadIdx.x] = sum;
        __syncthreads();
        if (group == 0)
            for (int x = 1; x < groups; x++) sum += so[threadIdx.x + x * lanes];
    }
    const float total = stat[mine];
    if (group == 0 && d < D && (int64_t)blockIdx.x * ROWS + mine < rows)
        *reinterpret_cast<f32x4_a4*>(a.out + bt * a.ldo + (int64_t)h * D + d) = total == 0.0f ? f32x4{0, 0, 0, 0} : sum / total;
}

struct TreeSplit {
    int tiles, split, parts;   // 16 rows each that a wave takes; positions of a part; parts
};
// How a call's rows and positions are shared out.  Workgroups enough to fill the card once where each is long (two tiles of rows a wave,
// two workgroups a CU: 512; 64 nodes over 50001 positions take 148 us, and 159 with 1024, which leave twice the parts to join), and
// some four times where a wave takes one and requests are ragged (2048: batches of 16 in f16 and 32 in 8 bits 175 and 161 us; 1024:
// 192 and 164, 4096: 207 and 170).  All by max_len, which the host knows, and not by the lengths: with a max_len of 131072 the same four
// calls (one of 8 nodes, one of 64, 16 and 32 requests) have longer parts for fewer workgroups and take 29, 225, 535 and 371 us in place
// of 13, 145, 173 and 159.
static int tiles_of(int R, int dim) { return R <= 64 || dim > 128 ? 1 : 2; }
static int64_t columns_of(int seqs, int heads, int R, int tiles) {
    return (int64_t)seqs * heads * ((R + 64 * tiles - 1) / (64 * tiles));
}
static int workgroups_of(int tiles) { return tiles == 2 ? 512 : 2048; }
static TreeSplit split_of(int seqs, int heads, int group, int dim, int T, int max_len) {
    TreeSplit s;
    const int R = T * group;
    s.tiles = tiles_of(R, dim);
    const int64_t columns = columns_of(seqs, heads, R, s.tiles);
    const int64_t want = (workgroups_of(s.tiles) + columns - 1) / columns;
    int64_t split = (max_len + want - 1) / want;
    if (split < (max_len + TJ_MOST - 1) / TJ_MOST) split = (max_len + TJ_MOST - 1) / TJ_MOST;
    split = (split + 31) / 32 * 32;
    s.split = (int)split;
    s.parts = (int)((max_len + split - 1) / split);
    return s;
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

static size_t bytes_of(size_t rows, int dim, int64_t parts) {
    return parts == 1 ? 256 : up256(rows * parts * dim * 4) + up256(rows * parts * sizeof(AttnMl));
}

size_t attn_tree_bytes(int seqs, int heads, int group, int dim, int T, int max_len) {
    return bytes_of((size_t)seqs * T * heads * group, dim, split_of(seqs, heads, group, dim, T, max_len).parts);
}

// The most that any call needs of up to so many requests, nodes and positions, whatever the key-value heads.  Parts come up to
// the least of what the workgroups ask for and the tiles of max_len, and some shorter max_len meets that; several requests that share the
// workgroups may need less than fewer do, and past as many as the workgroups each has one part.
size_t attn_tree_workspace(int seqs, int q_heads, int dim, int T, int max_len) {
    size_t most = 256;
    const int64_t tiles_long = (max_len + 31) / 32;
    for (int heads = 1; heads <= q_heads; heads++)
        for (int t = 1; t <= T && q_heads % heads == 0; t++) {
            const int R = t * (q_heads / heads), tiles = tiles_of(R, dim), all = workgroups_of(tiles);
            for (int b = 1; b <= seqs; b++) {
                const int64_t columns = columns_of(b, heads, R, tiles), want = (all + columns - 1) / columns;
                const size_t n = bytes_of((size_t)b * t * q_heads, dim, want < tiles_long ? want : tiles_long);
                most = n > most ? n : most;
                if (want == 1) break;
            }
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
    // few parts: a row's threads are its lanes alone, and several rows share a workgroup
    auto go = [&](auto kernel, int each) {
        const size_t lds = ((size_t)each * a.parts + 3) / 4 * 16 + (256 / each > lanes ? 4096 : 0);
        hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + each - 1) / each)), dim3(256), lds, s, a, lanes);
    };
    if (a.parts > 16) go(k_attn_tree_join<1>, 1);
    else if (lanes == 64) go(k_attn_tree_join<4>, 4);
    else if (lanes == 32) go(k_attn_tree_join<8>, 8);
    else go(k_attn_tree_join<16>, 16);
}

}  // namespace kq
