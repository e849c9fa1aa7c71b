// Attention of each request's last tokens over a paged key-value cache (include/kq.h: kq_attn_paged): the join of the chunks'
// parts that attn_paged.h's kernels leave.
#include <math.h>

#include "attn_paged.h"

namespace kq {

// One workgroup per row and 32 of its values: 32 groups of 8 lanes take every 32nd chunk, then the groups are added as a
// tree: a row's result depends on its number of chunks alone.
__global__ void __launch_bounds__(256) k_attn_join(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 so[4][8];
    __shared__ float sl[4], sm[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = a.kv.dim;
    const int b = blockIdx.x / a.T, h = blockIdx.y, d = 32 * blockIdx.z + 4 * (tid & 7);
    const int len = min(a.lens[b], a.max_len), n = len <= 0 ? 0 : (len + AT_CHUNK - 1) / AT_CHUNK;
    const int64_t row = ((int64_t)blockIdx.x * a.q_heads + h) * a.chunks;
    float top = -INFINITY;
    for (int c = tid; c < n; c += 256) top = fmaxf(top, a.pml[row + c].m);
    for (int w = 32; w; w >>= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
    if (lane == 0) sm[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll 8
    for (int c = tid >> 3; c < n; c += 32) {
        const AttnMl ml = a.pml[row + c];
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.po + (row + c) * D + (d < D ? d : 0));
        const float k = ml.l != 0.0f ? __builtin_amdgcn_exp2f(ml.m - top) : 0.0f;   // 0: the row saw nothing (a NaN counts)
        sum += x * k;
        total += ml.l * k;
    }
    for (int w = 8; w < 64; w <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i] += __shfl_xor(sum[i], w, 64);
        total += __shfl_xor(total, w, 64);
    }
    if (lane < 8) so[wave][lane] = sum;
    if (lane == 0) sl[wave] = total;
    __syncthreads();
    if (tid >= 8 || d >= D) return;
    sum = (so[0][tid] + so[1][tid]) + (so[2][tid] + so[3][tid]);
    total = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    *reinterpret_cast<f32x4_a4*>(a.out + (int64_t)blockIdx.x * a.ldo + (int64_t)h * D + d) =
        total == 0.0f ? f32x4{0, 0, 0, 0} : sum / total;
}

static int chunks_of(int max_len) { return max_len / AT_CHUNK + (max_len % AT_CHUNK != 0); }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t attn_paged_workspace(int seqs, int q_heads, int dim, int T, int max_len) {
    const size_t parts = (size_t)seqs * T * q_heads * chunks_of(max_len);
    return max_len <= AT_CHUNK ? 256 : up256(parts * dim * 4) + up256(parts * sizeof(AttnMl));
}

void launch_attn_paged(const AttnArgs& args, hipStream_t s) {
    AttnArgs a = args;
    a.page_shift = __builtin_ctz((unsigned)a.kv.page_size);
    a.chunks = chunks_of(a.max_len);
    a.joined = a.chunks > 1;
    const size_t parts = (size_t)a.table.seqs * a.T * a.q_heads * a.chunks;
    a.po = reinterpret_cast<float*>(a.ws);
    a.pml = reinterpret_cast<AttnMl*>(a.ws + up256(parts * a.kv.dim * 4));
    if (a.kv.type == KQ_KV_F16) launch_attn_part<KvF16>(a, s);
    else if (a.kv.type == KQ_KV_BF16) launch_attn_part<KvBf16>(a, s);
    else launch_attn_part<KvI8>(a, s);
    if (a.joined)
        hipLaunchKernelGGL(k_attn_join, dim3(a.table.seqs * a.T, a.q_heads, (a.kv.dim + 31) / 32), dim3(256), 0, s, a);
}

}  // namespace kq
