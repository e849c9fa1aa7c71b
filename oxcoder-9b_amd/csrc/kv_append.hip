// Append to a paged key-value cache: rotate the new tokens' queries and keys, store keys and values
// (include/kq.h: kq_kv_append).
//
// One thread holds 8 values of a head: the 4 pairs (i, i + rot/2) or (2i, 2i + 1) that it rotates, or, past the
// rotated part, 8 neighbours.  A head takes the next power of two of dim / 8 lanes, so the maximum that an
// 8-bit cache's scale needs is a few lane exchanges.  Every value is read once and written once; the kernel is
// bound by memory from some thousand tokens on (2 x 2048 tokens of 32 + 8 heads of 128 into bf16: 186 MB in 36 us, 5.2 TB/s; a large
// copy reaches 4.8) and by the launch and three dependent loads (position, page, data) below (one token 2.7 us).
// 8-bit codes divide by the scale as IEEE does, ten instructions a value that hide under the loads (3 x 341 tokens 12 us, 44 MB).
#include "kv_device.h"

namespace kq {

// 4 floats at p; V4: p is 16-byte aligned.
template <bool V4>
__device__ __forceinline__ f32x4 ld4f(const float* p) {
    if constexpr (V4) return *reinterpret_cast<const f32x4*>(p);
    return *reinterpret_cast<const f32x4_a4*>(p);
}

// Two groups of 4 neighbouring values, the first at `at` of the head and the second at `at + gap`.
template <class KV>
__device__ __forceinline__ void store8(typename KV::T* p, int gap, f32x4 a, f32x4 b, float scale) {
    if constexpr (KV::id == KQ_KV_I8) {
        auto code = [&](float x) {
            const float c = scale > 0.0f ? rintf(x / scale) : 0.0f;
            return (uint32_t)(int)fminf(fmaxf(c, -127.0f), 127.0f) & 0xffu;
        };
        auto pack = [&](f32x4 x) { return code(x.x) | code(x.y) << 8 | code(x.z) << 16 | code(x.w) << 24; };
        *reinterpret_cast<uint32_t*>(p) = pack(a);
        *reinterpret_cast<uint32_t*>(p + gap) = pack(b);
    } else {
        auto half = [&](float x) -> uint32_t {
            if constexpr (KV::id == KQ_KV_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
            else return bf16_rne(x);
        };
        auto pack = [&](f32x4 x) { return u32x2{half(x.x) | half(x.y) << 16, half(x.z) | half(x.w) << 16}; };
        *reinterpret_cast<u32x2*>(p) = pack(a);
        *reinterpret_cast<u32x2*>(p + gap) = pack(b);
    }
}

template <class KV, bool V4>
__global__ void __launch_bounds__(256) k_kv_append(AppendArgs a, int lanes) {
    const int D = a.kv.dim, H = a.q_heads + 2 * a.kv.heads;
    const int per = 256 / lanes;                              // heads per workgroup
    const int64_t head = (int64_t)blockIdx.x * per + threadIdx.x / lanes;
    const int i = threadIdx.x % lanes;                        // group of 8 values in the head
    if (head >= (int64_t)a.N * H) return;                     // whole lane groups end together
    const int n = (int)(head / H), h = (int)(head % H);
    const int pos = a.pos[n], seq = a.seq[n];
    if (seq < 0 || seq >= a.table.seqs || pos < 0 || pos >= a.table.cap || (a.rot && pos >= a.rope_rows)) return;
    const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv.heads;
    const int kh = is_q ? 0 : h - a.q_heads - (is_v ? a.kv.heads : 0);
    const float* x = is_q ? a.q + (int64_t)n * a.ldq + (int64_t)h * D
                          : (is_v ? a.v + (int64_t)n * a.ldv : a.k + (int64_t)n * a.ldk) + (int64_t)kh * D;
    const int rot = is_v ? 0 : a.rot, half = rot / 2;
    const bool live = 8 * i < D, turns = 8 * i < rot;
    // where the group's two quarters lie in the head
    const int at = turns && !a.interleaved ? 4 * i : 8 * i, gap = turns && !a.interleaved ? half : 4;
    f32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (live) {
        lo = ld4f<V4>(x + at);
        hi = ld4f<V4>(x + at + gap);
    }
    if (live && turns) {
        const float* r = a.rope + (int64_t)pos * a.rot + 4 * i;
        const f32x4 c = ld4f<V4>(r), s = ld4f<V4>(r + half);
        if (a.interleaved) {
            const f32x4 l = lo, m = hi;
            lo = f32x4{l.x * c.x - l.y * s.x, l.y * c.x + l.x * s.x, l.z * c.y - l.w * s.y, l.w * c.y + l.z * s.y};
            hi = f32x4{m.x * c.z - m.y * s.z, m.y * c.z + m.x * s.z, m.z * c.w - m.w * s.w, m.w * c.w + m.z * s.w};
        } else {
            const f32x4 l = lo;
            lo = l * c - hi * s;
            hi = hi * c + l * s;
        }
    }
    if (is_q) {
        if (!live) return;
        float* y = a.q_out + (int64_t)n * a.ldqo + (int64_t)h * D + at;
        if constexpr (V4) {
            *reinterpret_cast<f32x4*>(y) = lo;
            *reinterpret_cast<f32x4*>(y + gap) = hi;
        } else {
            *reinterpret_cast<f32x4_a4*>(y) = lo;
            *reinterpret_cast<f32x4_a4*>(y + gap) = hi;
        }
        return;
    }
    const int page = a.table.pages[(int64_t)seq * a.table.ld + pos / a.kv.page_size];
    if (page < 0 || page >= a.kv.pages) return;
    const int off = pos & (a.kv.page_size - 1);
    float scale = 0.0f;
    if constexpr (KV::id == KQ_KV_I8) {
        float m = fmaxf(fmaxf(fabsf(lo.x), fabsf(lo.y)), fmaxf(fabsf(lo.z), fabsf(lo.w)));
        m = fmaxf(m, fmaxf(fmaxf(fabsf(hi.x), fabsf(hi.y)), fmaxf(fabsf(hi.z), fabsf(hi.w))));
        for (int w = lanes >> 1; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
        scale = m * (1.0f / 127.0f);
        if (i == 0)
            (is_v ? a.kv.v_scale : a.kv.k_scale)[page * a.kv.scale_page_stride + kh * a.kv.scale_head_stride +
                                                 off * a.kv.scale_pos_stride] = scale;
    }
    if (live)
        store8<KV>(static_cast<typename KV::T*>(is_v ? a.kv.v : a.kv.k) + page * a.kv.page_stride +
                       kh * a.kv.head_stride + off * a.kv.pos_stride + at,
                   gap, lo, hi, scale);
}

void launch_kv_append(const AppendArgs& a, hipStream_t s) {
    int lanes = 2;
    while (lanes * 8 < a.kv.dim) lanes *= 2;
    const int per = 256 / lanes;
    const int64_t heads = (int64_t)a.N * (a.q_heads + 2 * a.kv.heads);
    const dim3 grid((unsigned)((heads + per - 1) / per));
    auto al = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0; };
    const bool v4 = al(a.k, a.ldk) && al(a.v, a.ldv) && (!a.q_heads || (al(a.q, a.ldq) && al(a.q_out, a.ldqo))) &&
                    (!a.rot || al(a.rope, 0));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, lanes); };
    if (a.kv.type == KQ_KV_F16) v4 ? go(k_kv_append<KvF16, true>) : go(k_kv_append<KvF16, false>);
    else if (a.kv.type == KQ_KV_BF16) v4 ? go(k_kv_append<KvBf16, true>) : go(k_kv_append<KvBf16, false>);
    else v4 ? go(k_kv_append<KvI8, true>) : go(k_kv_append<KvI8, false>);
}

}  // namespace kq
