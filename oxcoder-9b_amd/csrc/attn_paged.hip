// Attention of each request's last tokens over a paged key-value cache (include/kq.h: kq_attn_paged).
#include "kv_device.h"

namespace kq {

// One workgroup per row; its waves take every fourth position, a lane up to 4 values of the head.
template <class KV>
__global__ void __launch_bounds__(256) k_attn_rows(AttnArgs a) {
    __shared__ float sm[4], sl[4], so[4][256];
    const int D = a.kv.dim, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.x, b = blockIdx.y / a.T, t = blockIdx.y % a.T;
    const int len = min(min(a.lens[b], a.max_len), a.table.cap), upto = len - a.T + 1 + t;
    const int kh = h / (a.q_heads / a.kv.heads);
    float q[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
    for (int i = 0; i < 4; i++)
        q[i] = lane + 64 * i < D ? a.q[(int64_t)blockIdx.y * a.ldq + (int64_t)h * D + lane + 64 * i] * a.scale : 0.0f;
    for (int p = wave; p < upto; p += 4) {
        const int page = a.table.pages[(int64_t)b * a.table.ld + p / a.kv.page_size];
        if (page < 0 || page >= a.kv.pages) continue;
        const int off = p & (a.kv.page_size - 1);
        const int64_t at = page * a.kv.page_stride + kh * a.kv.head_stride + off * a.kv.pos_stride;
        float ks = 1, vs = 1;
        if constexpr (KV::id == KQ_KV_I8) {
            const int64_t sat = page * a.kv.scale_page_stride + kh * a.kv.scale_head_stride + off * a.kv.scale_pos_stride;
            ks = a.kv.k_scale[sat];
            vs = a.kv.v_scale[sat];
        }
        auto val = [&](const void* base, int i) {
            const typename KV::T x = static_cast<const typename KV::T*>(base)[at + lane + 64 * i];
            if constexpr (KV::id == KQ_KV_BF16) return __builtin_bit_cast(float, (uint32_t)x << 16);
            else return (float)x;
        };
        float s = 0;
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < D) s += q[i] * val(a.kv.k, i);
        for (int w = 32; w; w >>= 1) s += __shfl_xor(s, w, 64);
        s *= ks;
        const float mn = fmaxf(m, s), keep = mn == m ? 1.0f : expf(m - mn), e = expf(s - mn);
        for (int i = 0; i < 4; i++) o[i] = o[i] * keep + (lane + 64 * i < D ? e * vs * val(a.kv.v, i) : 0.0f);
        l = l * keep + e;
        m = mn;
    }
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
    for (int i = 0; i < 4; i++) so[wave][lane + 64 * i] = o[i];
    __syncthreads();
    if ((int)threadIdx.x >= D) return;
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float sum = 0, val = 0;
    for (int w = 0; w < 4; w++) {
        const float f = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - top);
        sum += sl[w] * f;
        val += so[w][threadIdx.x] * f;
    }
    a.out[(int64_t)blockIdx.y * a.ldo + (int64_t)h * D + threadIdx.x] = sum == 0 ? 0.0f : val / sum;
}

size_t attn_paged_workspace(int, int, int, int, int) { return 256; }

void launch_attn_paged(const AttnArgs& a, hipStream_t s) {
    const dim3 grid(a.q_heads, a.table.seqs * a.T);
    if (a.kv.type == KQ_KV_F16) hipLaunchKernelGGL(k_attn_rows<KvF16>, grid, dim3(256), 0, s, a);
    else if (a.kv.type == KQ_KV_BF16) hipLaunchKernelGGL(k_attn_rows<KvBf16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_attn_rows<KvI8>, grid, dim3(256), 0, s, a);
}

}  // namespace kq
