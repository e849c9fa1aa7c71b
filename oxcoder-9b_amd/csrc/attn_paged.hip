// Attention of each request's last tokens over a paged key-value cache (include/kq.h: kq_attn_paged): the join of the chunks'
// parts that attn_paged.h's kernels leave.
#include <math.h>

#include "attn_paged.h"

namespace kq {

// One workgroup per row and 32 N of its values: 32 groups of 8 lanes take every 32nd pair of chunks, in the steps of
// the workgroup that had both where there was one; then the groups are added as a tree: a row's result depends on its
// number of chunks alone.
template <int N, bool PAIRED>
__global__ void __launch_bounds__(256) k_attn_join(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) f32x4 so[4][N][8];
    __shared__ float sl[4], sm[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = a.kv.dim;
    const int b = blockIdx.x / a.T, h = blockIdx.y, G = a.group, d = 32 * N * blockIdx.z + 4 * (tid & 7);
    const int len = min(a.lens[b], a.max_len), n = len <= 0 ? 0 : (len + AT_CHUNK - 1) / AT_CHUNK, pairs = (n + 1) / 2;
    const int64_t row = (((int64_t)b * a.kv.heads + h / G) * a.T * G + blockIdx.x % a.T * G + h % G) * a.parts;
    float top = -INFINITY;
    for (int c = tid; c < (PAIRED ? pairs : n); c += 256) top = fmaxf(top, a.pml[row + c].m);
    for (int w = 32; w; w >>= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
    if (lane == 0) sm[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    f32x4 sum[N] = {};
    float total = 0.0f;
    auto load = [&](int64_t part, f32x4 (&x)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = *reinterpret_cast<const f32x4*>(a.po + part * D + (d + 32 * i < D ? d + 32 * i : 0));
    };
    auto add = [&](AttnMl ml, const f32x4 (&x)[N]) {
        const float k = ml.l != 0.0f ? __builtin_amdgcn_exp2f(ml.m - top) : 0.0f;   // 0: the row saw nothing (a NaN counts)
#pragma unroll
        for (int i = 0; i < N; i++) sum[i] += x[i] * k;
        total += ml.l * k;
    };
    if constexpr (PAIRED) {
#pragma unroll 8 / N
        for (int c = tid >> 3; c < pairs; c += 32) {
            f32x4 x[N];
            load(row + c, x);
            add(a.pml[row + c], x);
        }
    } else {
#pragma unroll 4 / N
        for (int c = tid >> 3; c < pairs; c += 32) {
            const int64_t p0 = row + 2 * c, p1 = 2 * c + 1 < n ? p0 + 1 : p0;
            const AttnMl m0 = a.pml[p0];
            AttnMl m1 = a.pml[p1];
            f32x4 x[N], y[N];
            load(p0, x);
            load(p1, y);
            if (p1 != p0) {
                const AtPair p = at_pair(m0, m1);
#pragma unroll
                for (int i = 0; i < N; i++) x[i] = x[i] * p.k0 + y[i] * p.k1;
                m1 = AttnMl{p.top, p.l};
            }
            add(m1, x);
        }
    }
#pragma unroll
    for (int w = 8; w < 64; w <<= 1) {
#pragma unroll
        for (int i = 0; i < 4 * N; i++) sum[i >> 2][i & 3] += __shfl_xor(sum[i >> 2][i & 3], w, 64);
        total += __shfl_xor(total, w, 64);
    }
    if (lane < 8)
#pragma unroll
        for (int i = 0; i < N; i++) so[wave][i][lane] = sum[i];
    if (lane == 0) sl[wave] = total;
    __syncthreads();
    const int i = tid >> 3, at = 32 * N * blockIdx.z + 4 * tid;
    if (i >= N || at >= D) return;
    const f32x4 all = (so[0][i][tid & 7] + so[1][i][tid & 7]) + (so[2][i][tid & 7] + so[3][i][tid & 7]);
    total = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    *reinterpret_cast<f32x4_a4*>(a.out + (int64_t)blockIdx.x * a.ldo + (int64_t)h * D + at) =
        total == 0.0f ? f32x4{0, 0, 0, 0} : all / total;
}

static int chunks_of(int max_len) { return max_len / AT_CHUNK + (max_len % AT_CHUNK != 0); }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t attn_paged_workspace(int seqs, int q_heads, int dim, int T, int max_len) {
    const size_t parts = (size_t)seqs * T * q_heads * chunks_of(max_len);
    return max_len <= AT_CHUNK ? 256 : up256(parts * dim * 4) + up256(parts * sizeof(AttnMl));
}

void launch_attn_paged(const AttnArgs& args, hipStream_t s) {
    AttnArgs a = args;
    a.scale *= 1.44269504088896341f;                           // scores in powers of 2
    a.group = a.q_heads / a.kv.heads;
    a.page_shift = __builtin_ctz((unsigned)a.kv.page_size);
    a.chunks = chunks_of(a.max_len);
    a.joined = a.chunks > 1;
    // Where that leaves six workgroups a CU, a workgroup takes two chunks, the second's first step in flight while it ends the first, and
    // leaves one part for both; four chunks where that leaves sixteen.  One, two, four chunks a workgroup, us, requests
    // of 4096 positions with 8 heads of 128 values, by the chunks of all: bf16 640 21, 25, 26; 1536 37, 38, 42; 2304 60, 59, 63; 3072
    // 80, 74, 74; 4608 118, 109, 113; 12288 310, 279, 279; 25600 641, 575, 576; 8-bit 640 19, 22, 29; 1536 31, 30, 36; 2304 41,
    // 42, 45; 3072 51, 49, 47; 4608 81, 76, 78; 12288 213, 197, 192; 25600 432, 398, 380.
    const int64_t all = (int64_t)a.chunks * a.kv.heads * a.table.seqs * ((a.T * a.group + 15) / 16), cus = device_cus();
    a.paired = a.joined && all >= 12 * cus;
    a.parts = a.paired ? (a.chunks + 1) / 2 : a.chunks;
    a.groups = all >= 64 * cus ? (a.parts + 1) / 2 : a.parts;
    if (a.groups > 65535) a.groups = 65535;                    // a workgroup goes on until no chunk is left
    const size_t parts = (size_t)a.table.seqs * a.T * a.q_heads * a.parts;
    a.po = reinterpret_cast<float*>(a.ws);
    a.pml = reinterpret_cast<AttnMl*>(a.ws + up256(parts * a.kv.dim * 4));
    if (a.kv.type == KQ_KV_F16) launch_attn_part<KvF16>(a, s);
    else if (a.kv.type == KQ_KV_BF16) launch_attn_part<KvBf16>(a, s);
    else launch_attn_part<KvI8>(a, s);
    if (!a.joined) return;
    // rows enough for the chip: four times fewer workgroups, that scan a row's maxima once for 128 values (512 rows of 20 chunks and
    // 256 values 7.4 -> 5 us; the 32 rows of 391 chunks 8 us with 32 values each, 13 us with 128)
    const int64_t rows = (int64_t)a.table.seqs * a.T * a.q_heads;
    const bool wide = rows >= device_cus();
    const dim3 grid(a.table.seqs * a.T, a.q_heads, wide ? (a.kv.dim + 127) / 128 : (a.kv.dim + 31) / 32);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (a.paired) wide ? go(k_attn_join<4, true>) : go(k_attn_join<1, true>);
    else wide ? go(k_attn_join<4, false>) : go(k_attn_join<1, false>);
}

}  // namespace kq
