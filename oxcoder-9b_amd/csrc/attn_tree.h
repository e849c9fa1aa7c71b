// Attention of trees of drafted tokens over a paged key-value cache (include/kq.h: kq_attn_tree), the part that reads the cache
// (attn_tree.hip joins the parts).
//
//   out = sum_p e_p v_p / sum_p e_p,   e_p = 2^(x_p - m),   x_p = scale log2(e) q.k_p,   m = max x_p over what the row sees
//
// A tree's rows (nodes x query heads of a key-value head) are many, so here they share what a workgroup reads: it takes a
// split of the positions for 16 NT rows of each of its four waves, and every key and value goes once through LDS for
// all of them, in tiles of 32 positions.  A wave's step is such a tile, with 16x16x32 bf16 MFMAs:
//   S^T [position][row] = K [position][d] Q^T [d][row],   O^T [d][row] += V^T [d][position] E^T [position][row].
// The result layout of the first (lane: row lane % 16, positions 4 (lane / 16) + 0..3 of a 16) is the operand layout of the
// second for the order of positions in which V^T is read, by transposing LDS loads of 4 positions at a time.
//
// q and e are fp32, held in three bf16 parts of 8 bits each truncated from what the one before left: their products with
// bf16 values are exact, and sums fp32.  8-bit codes are bf16 values; an f16 value is the sum of two, its top 8 bits and the 3
// that they leave, of which the second meets the first two parts of q and e (the third would add below 2^-24 of the product).
#pragma once
#include "attn_paged.h"

namespace kq {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The positions of a request that are there: those ahead of its tree, and T more.
__device__ __forceinline__ int tree_length(const AttnArgs& a, int base) {
    return base < 0 ? 0 : min(min(base, a.max_len) + a.T, a.max_len);
}

// Both elements' three parts, the first element in the low half.
__device__ __forceinline__ void split3(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    auto cut = [](float a) { return fbits(ubits(a) & 0xffff0000u); };
    const float rx = x - cut(x), ry = y - cut(y);
    p0 = hi_halves(ubits(x), ubits(y));
    p1 = hi_halves(ubits(rx), ubits(ry));
    p2 = hi_halves(ubits(rx - cut(rx)), ubits(ry - cut(ry)));
}

// Eight f16 values as the sums of two bf16 values; an infinity or NaN stays in the first.
__device__ __forceinline__ void f16_pair(u32x4 raw, u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float x = f16_lo(raw[j]), y = f16_hi(raw[j]);
        const float cx = fbits(ubits(x) & 0xffff0000u), cy = fbits(ubits(y) & 0xffff0000u);
        hi[j] = hi_halves(ubits(x), ubits(y));
        const uint32_t r = hi_halves(ubits(x - cx), ubits(y - cy));
        lo[j] = r;
    }
    // inf - inf and NaN - NaN are NaN: the second part of such a value is 0
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if ((hi[j] & 0x7f80u) == 0x7f80u) lo[j] &= 0xffff0000u;
        if ((hi[j] >> 16 & 0x7f80u) == 0x7f80u) lo[j] &= 0xffffu;
    }
}

__device__ __forceinline__ f32x4 mma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight 16-bit values of exponent bits E, 0 in the place of infinities and NaN.
template <uint32_t E>
__device__ __forceinline__ u32x4 finite(u32x4 x) {
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] &= ((x[j] & E) == E ? 0u : 0xffffu) | ((x[j] >> 16 & E) == E ? 0u : 0xffff0000u);
    return x;
}

// ND: 16ths of the head size, which may be less (the rest counts as 0).
template <class KV, int ND, int NT>
struct TreeAttn {
    static constexpr bool I8 = KV::id == KQ_KV_I8, F16 = KV::id == KQ_KV_F16;
    static constexpr int D = 16 * ND, EB = I8 ? 1 : 2, QS = ND / 2, P = 32;
    static constexpr int PLANES = F16 ? 2 : 1;
    static constexpr int ROW = 2 * D + 16;                 // bytes of a position in LDS: rows fall on other banks each
    static constexpr int PLANE = P * ROW, TILE = 2 * PLANES * PLANE;
    static constexpr int NBUF = 2 * TILE <= 72 * 1024 ? 2 : 1;
    static constexpr int UNITS = D * EB / 16;              // 16-byte pieces of a position
    static constexpr int MINE = 8;                         // positions that a wave fetches
    static constexpr int PER = (MINE * UNITS + 63) / 64;   // pieces of a lane
    static constexpr bool AHEAD = ND < 16 && NT == 1;      // fragments are read ahead of their use, where registers are left
    static constexpr size_t LDS = (size_t)TILE * NBUF;
};

template <class KV, int ND, int NT>
__global__ void __launch_bounds__(256, ND * NT <= 4 ? 4 : ND * NT <= 8 ? 3 : 2) k_attn_tree(AttnArgs a) {
    typedef TreeAttn<KV, ND, NT> A;
    extern __shared__ __attribute__((aligned(16))) uint8_t tiles[];
    __shared__ uint32_t there[A::NBUF][4];
    __shared__ __attribute__((aligned(16))) float scales[A::NBUF][2][A::I8 ? A::P : 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int kh = blockIdx.x % a.kv.heads, rb = blockIdx.x / a.kv.heads, b = blockIdx.y, z = blockIdx.z;
    const int G = a.group, R = a.T * G, D = a.kv.dim;
    const int base = __builtin_amdgcn_readfirstlane(a.lens[b]), len = tree_length(a, base);
    const int from = z * a.split, to = min(len, from + a.split);
    if (from >= len && z) return;                              // the join knows the splits that are there
    const int row0 = 16 * NT * (4 * rb + wave);              // the wave's first
    const bool idle = row0 >= R;

    // what the rows see of the tree, and what any row does
    const uint64_t* seen = a.seen + (int64_t)b * a.T;
    const uint64_t word = lane < a.T ? seen[lane] : 0;
    uint32_t lo = (uint32_t)word, hi = (uint32_t)(word >> 32);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) lo |= of_lane(lane ^ i, lo), hi |= of_lane(lane ^ i, hi);
    const uint64_t some = (uint64_t)__builtin_amdgcn_readfirstlane(hi) << 32 | __builtin_amdgcn_readfirstlane(lo);
    // (Read again where it is needed, and the thread's place below taken anew for each tile: neither is held.)
    auto nodes_of = [&](int n) __attribute__((always_inline)) {
        int row = row0 + 16 * n + (lane & 15);
        asm volatile("" : "+v"(row));
        return seen[min(row / G, a.T - 1)];
    };
    auto here = [&]() __attribute__((always_inline)) {
        int i = lane;
        asm volatile("" : "+v"(i));
        return i;
    };

    // Keys past the head's size stay 0 from here on.
    if (D < A::D)
        for (int i = tid; i < A::NBUF * A::PLANES * A::P; i += 256) {
            uint8_t* row = tiles + i / (A::PLANES * A::P) * A::TILE + i % (A::PLANES * A::P) * A::ROW;
            for (int d = D; d < A::D; d += 8) *reinterpret_cast<u32x4*>(row + 2 * d) = u32x4{0, 0, 0, 0};
        }

    // Fetching: lane i of a wave looks after the place of position MINE wave + i of the tile, and holds PER pieces.
    const int32_t* table = a.table.pages + (int64_t)b * a.table.ld;
    const uint8_t* kb = static_cast<const uint8_t*>(a.kv.k) + (int64_t)kh * a.kv.head_stride * A::EB;
    const uint8_t* vb = static_cast<const uint8_t*>(a.kv.v) + (int64_t)kh * a.kv.head_stride * A::EB;
    auto entry = [&](int first) __attribute__((always_inline)) {
        return table[min(first + A::MINE * wave + here() % A::MINE, a.table.cap - 1) >> a.page_shift];
    };
    u32x4 kreg[A::PER], vreg[A::PER];
    uint32_t ok_bits = 0;
    bool wild = false;                                         // values that are not finite count as 0 (below)
    float ks = 0.0f, vs = 0.0f;
    auto fetch = [&](int first, int page) __attribute__((always_inline)) {
        const int lane = here(), p = first + A::MINE * wave + lane % A::MINE, node = p - base;
        const bool ok = p < to && (unsigned)page < (unsigned)a.kv.pages && (node < 0 || (node < 64 && (some >> node & 1u)));
        const int off = p & (a.kv.page_size - 1);
        const int64_t at = ok ? (page * a.kv.page_stride + off * a.kv.pos_stride) * A::EB : 0;
        ok_bits = (uint32_t)__ballot(ok) & ((1u << A::MINE) - 1u);
        if constexpr (A::I8) {
            const int64_t e = page * a.kv.scale_page_stride + kh * a.kv.scale_head_stride + off * a.kv.scale_pos_stride;
            ks = ok ? a.kv.k_scale[e] : 0.0f;
            vs = ok ? a.kv.v_scale[e] : 0.0f;
        }
        const uint32_t at_lo = (uint32_t)at, at_hi = (uint32_t)(at >> 32);
#pragma unroll
        for (int i = 0; i < A::PER; i++) {
            const int u = 64 * i + lane, pos = u / A::UNITS % A::MINE, col = u % A::UNITS;
            const int64_t place = (int64_t)((uint64_t)of_lane(pos, at_hi) << 32 | of_lane(pos, at_lo)) + 16 * col;
            const bool live = ok_bits >> pos & 1u && 16 * col < D * A::EB;
            u32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
            if (live) {
                k = *reinterpret_cast<const u32x4*>(kb + place);
                v = *reinterpret_cast<const u32x4*>(vb + place);
            }
            kreg[i] = k, vreg[i] = v;
        }
    };
    auto put = [&](int buf) __attribute__((always_inline)) {
        const int lane = here(), mine = A::MINE * wave + lane % A::MINE;
        uint8_t* kt = tiles + buf * A::TILE + A::MINE * wave * A::ROW;
        uint8_t* vt = kt + A::PLANES * A::PLANE;
#pragma unroll
        for (int i = 0; i < A::PER; i++) {
            const int u = 64 * i + lane, pos = u / A::UNITS, col = u % A::UNITS;
            u32x4 k = kreg[i], v = vreg[i];
            const bool live = (A::MINE * A::UNITS % 64 == 0 || pos < A::MINE) && 16 * col < D * A::EB;
            uint8_t *kp = kt + pos * A::ROW + 16 / A::EB * 2 * col, *vp = vt + pos * A::ROW + 16 / A::EB * 2 * col;
            if constexpr (A::I8) {
                const u32x4 k0 = code_bf16(k.x, k.y), k1 = code_bf16(k.z, k.w), v0 = code_bf16(v.x, v.y), v1 = code_bf16(v.z, v.w);
                if (live) {
                    *reinterpret_cast<u32x4*>(kp) = k0, *reinterpret_cast<u32x4*>(kp + 16) = k1;
                    *reinterpret_cast<u32x4*>(vp) = v0, *reinterpret_cast<u32x4*>(vp + 16) = v1;
                }
            } else {
                if (wild) v = finite<A::F16 ? 0x7c00u : 0x7f80u>(v);
                if constexpr (A::PLANES == 2) {
                    u32x4 kh, kl, vh, vl;
                    f16_pair(k, kh, kl);
                    f16_pair(v, vh, vl);
                    if (live) {
                        *reinterpret_cast<u32x4*>(kp) = kh, *reinterpret_cast<u32x4*>(kp + A::PLANE) = kl;
                        *reinterpret_cast<u32x4*>(vp) = vh, *reinterpret_cast<u32x4*>(vp + A::PLANE) = vl;
                    }
                } else if (live) {
                    *reinterpret_cast<u32x4*>(kp) = k;
                    *reinterpret_cast<u32x4*>(vp) = v;
                }
            }
        }
        if (lane == 0) there[buf][wave] = ok_bits;
        if (A::I8 && lane < A::MINE) scales[buf][0][mine] = ks, scales[buf][1][mine] = vs;
    };
    int page = entry(from);
    fetch(from, page);

    // q's parts, in powers of 2
    u32x4 qp[NT][A::QS][3];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int row = row0 + 16 * n + r, at = row < R ? row : 0;
        const float* q = a.q + ((int64_t)b * a.T + at / G) * a.ldq + (int64_t)(kh * G + at % G) * D;
#pragma unroll
        for (int s = 0; s < A::QS; s++) {
            const int d = 32 * s + 8 * g;
            f32x4 x[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                x[j] = d < D ? *reinterpret_cast<const f32x4_a4*>(q + d + 4 * j) : f32x4{0, 0, 0, 0};
                x[j] *= a.scale;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t p0, p1, p2;
                split_bf16(x[j >> 1][2 * (j & 1)], x[j >> 1][2 * (j & 1) + 1], p0, p1, p2);
                qp[n][s][0][j] = p0, qp[n][s][1][j] = p1, qp[n][s][2][j] = p2;
            }
        }
    }
    float m[NT], l[NT];
    f32x4 o[NT][ND];
    // Once, and once more where an infinity or NaN among the values left a sum that is not finite: it reached rows that do not see it
    // as 0 * inf.  Then such values count as 0, and are given to the rows that see them at the end.
    for (;;) {
    page = entry(from + A::P);
    put(0);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -INFINITY, l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[n][d] = f32x4{0, 0, 0, 0};
    }
    int buf = 0;
    for (int first = from; first < to; first += A::P) {
        const bool on = first + A::P < to;
        if (on) {
            fetch(first + A::P, page);
            page = entry(first + 2 * A::P);
        }
        if (!idle) {
            const uint8_t* kt = tiles + buf * A::TILE;
            const uint8_t* vt = kt + A::PLANES * A::PLANE;
            f32x4 acc[NT][2] = {};
            // a step of d for both 16 positions, the next one's on its way while it is multiplied (no more, which would cost
            // registers); the two in turn, so that no product waits for the one just before it
            u32x4 k[A::AHEAD ? 2 : 1][2][A::PLANES];
            auto key = [&](int i, u32x4 (&to)[2][A::PLANES]) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int j = 0; j < A::PLANES; j++)
                        to[t][j] = *reinterpret_cast<const u32x4*>(kt + (16 * t + r) * A::ROW + 64 * i + 16 * g + j * A::PLANE);
            };
            if (A::AHEAD) key(0, k[0]);
#pragma unroll
            for (int i = 0; i < A::QS; i++) {
                constexpr int B = A::AHEAD ? 1 : 0;
                if (!A::AHEAD) key(i, k[0]);
                else if (i + 1 < A::QS) key(i + 1, k[(i + 1) & B]);
                u32x4 kh[2], kl[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    kh[t] = k[i & B][t][0];
                    if constexpr (A::F16) kl[t] = k[i & B][t][A::PLANES - 1];
                }
                if constexpr (A::F16) {
#pragma unroll
                    for (int j = 1; j >= 0; j--)
#pragma unroll
                        for (int n = 0; n < 2 * NT; n++) acc[n >> 1][n & 1] = mma_bf16(kl[n & 1], qp[n >> 1][i][j], acc[n >> 1][n & 1]);
                }
#pragma unroll
                for (int j = 2; j >= 0; j--)
#pragma unroll
                    for (int n = 0; n < 2 * NT; n++) acc[n >> 1][n & 1] = mma_bf16(kh[n & 1], qp[n >> 1][i][j], acc[n >> 1][n & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (A::I8) {
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(&scales[buf][0][16 * t + 4 * g]);
#pragma unroll
                    for (int n = 0; n < NT; n++) acc[n][t] *= x;
                }
            }
            uint32_t ok = 0;                                   // the step's positions that are there
#pragma unroll
            for (int i = 0; i < 4; i++) ok |= there[buf][i] << A::MINE * i;
            ok = __builtin_amdgcn_readfirstlane(ok);
            const bool partly = ok != ~0u || first + 32 > base;
            uint32_t shown[NT];                                // bit i: the row sees position first + i
            if (partly) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const int at = first - base;                 // the first's place in the tree
                    const uint64_t nodes = nodes_of(n);
                    const uint64_t see = at >= 64 ? 0 : at >= 0 ? nodes >> at : at > -32 ? nodes << -at | ((1u << -at) - 1u) : ~0ull;
                    shown[n] = ok & (uint32_t)see;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (!(shown[n] >> (16 * (i >> 2) + 4 * g + (i & 3)) & 1u)) acc[n][i >> 2][i & 3] = -INFINITY;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, acc[n][i >> 2][i & 3]);
                top = fmaxf(m[n], xor32_max(xor16_max(top)));
                const float keep = m[n] == top ? 1.0f : __builtin_amdgcn_exp2f(m[n] - top);
                if (!__all(keep == 1.0f)) {
                    l[n] *= keep;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[n][d] *= keep;
                }
                m[n] = top;
                const float under = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = __builtin_amdgcn_exp2f(acc[n][i >> 2][i & 3] - under);
                    acc[n][i >> 2][i & 3] = x;
                    l[n] += x;
                }
            }
            {
                u32x4 ep[NT][3];
                f32x4 x[2];
                if constexpr (A::I8)
#pragma unroll
                    for (int t = 0; t < 2; t++) x[t] = *reinterpret_cast<const f32x4*>(&scales[buf][1][16 * t + 4 * g]);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float e0 = acc[n][j >> 1][2 * (j & 1)], e1 = acc[n][j >> 1][2 * (j & 1) + 1];
                        if constexpr (A::I8) {                 // a NaN stays one, a 0 takes no part
                            e0 = e0 == 0.0f ? e0 : e0 * x[j >> 1][2 * (j & 1)];
                            e1 = e1 == 0.0f ? e1 : e1 * x[j >> 1][2 * (j & 1) + 1];
                        }
                        uint32_t q0, q1, q2;
                        split3(e0, e1, q0, q1, q2);
                        ep[n][0][j] = q0, ep[n][1][j] = q1, ep[n][2][j] = q2;
                    }
                // four positions' values at a time, transposed: lane r's d, positions 4 g + 0..3 of each 16
                const uint8_t* at = vt + (4 * g + (r >> 2)) * A::ROW + 8 * (r & 3);
                auto value = [&](int d, u32x4 (&to)[2][A::PLANES]) __attribute__((always_inline)) {
#pragma unroll
                    for (int w = 0; w < 2; w++)
#pragma unroll
                        for (int j = 0; j < A::PLANES; j++) {
                            const uint8_t* from = at + j * A::PLANE + 32 * (d + w);
                            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)from));
                            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(from + 16 * A::ROW)));
                            to[w][j] = u32x4{x.x, x.y, y.x, y.y};
                        }
                };
                {
                    u32x4 v[A::AHEAD ? 2 : 1][2][A::PLANES];
                    constexpr int B = A::AHEAD ? 1 : 0;
                    if (A::AHEAD) value(0, v[0]);
#pragma unroll
                    for (int d = 0; d < ND; d += 2) {
                        if (!A::AHEAD) value(d, v[0]);
                        else if (d + 2 < ND) value(d + 2, v[((d >> 1) + 1) & B]);
                        u32x4 vh[2], vl[2];
#pragma unroll
                        for (int w = 0; w < 2; w++) {
                            const u32x4 raw = v[d >> 1 & B][w][0];
                            vh[w] = raw;
                            if constexpr (A::F16) vl[w] = v[d >> 1 & B][w][A::PLANES - 1];
                        }
                        if constexpr (A::F16) {
#pragma unroll
                            for (int j = 1; j >= 0; j--)
#pragma unroll
                                for (int n = 0; n < 2 * NT; n++) o[n >> 1][d + (n & 1)] = mma_bf16(vl[n & 1], ep[n >> 1][j], o[n >> 1][d + (n & 1)]);
                        }
#pragma unroll
                        for (int j = 2; j >= 0; j--)
#pragma unroll
                            for (int n = 0; n < 2 * NT; n++) o[n >> 1][d + (n & 1)] = mma_bf16(vh[n & 1], ep[n >> 1][j], o[n >> 1][d + (n & 1)]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
        if (A::NBUF == 1) __syncthreads();                     // the tile has been read
        if (on) put(A::NBUF == 2 ? buf ^ 1 : 0);
        __syncthreads();
        if (A::NBUF == 2) buf ^= 1;
    }

    if (A::I8 || wild) break;
    // 0 * x is 0 for every finite x
    f32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (16 * d < D) zero += o[n][d] * 0.0f;
    if (!__syncthreads_or(!idle && !(zero.x + zero.y + (zero.z + zero.w) == 0.0f))) break;
    wild = true;
    fetch(from, entry(from));
    }
    if (!A::I8 && wild && !idle) {
        uint64_t nodes[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) nodes[n] = nodes_of(n);
        {
            for (int p = from; p < to; p++) {
                const int page = __builtin_amdgcn_readfirstlane(table[p >> a.page_shift]);
                if ((unsigned)page >= (unsigned)a.kv.pages) continue;
                const uint8_t* at = vb + (page * a.kv.page_stride + (p & (a.kv.page_size - 1)) * a.kv.pos_stride) * A::EB + 8 * g;
                const int node = p - base;
#pragma unroll
                for (int d = 0; d < ND; d++)
                    if (16 * d < D) {
                        const u32x2 raw = *reinterpret_cast<const u32x2*>(at + 32 * d);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t half = i & 1 ? raw[i >> 1] >> 16 : raw[i >> 1] & 0xffffu;
                            const float v = A::F16 ? f16_lo(half) : fbits(half << 16);
#pragma unroll
                            for (int n = 0; n < NT; n++)
                                if (!(fabsf(v) < INFINITY) && (node < 0 || nodes[n] >> node & 1u)) o[n][d][i] += v;
                        }
                    }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        l[n] = xor32_sum(xor16_sum(l[n]));
        if (!nodes_of(n)) m[n] = -INFINITY, l[n] = 0.0f;          // no node: it has seen nothing
    }
    const int64_t part0 = (((int64_t)b * a.kv.heads + kh) * R) * a.parts + z;
    auto out_of = [&](int row) {
        return a.joined ? a.po + (part0 + (int64_t)row * a.parts) * D
                        : a.out + ((int64_t)b * a.T + row / G) * a.ldo + (int64_t)(kh * G + row % G) * D;
    };
    if (idle) return;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int row = row0 + 16 * n + r;
        if (row >= R) continue;
        if (a.joined && g == 0) a.pml[part0 + (int64_t)row * a.parts] = AttnMl{m[n], l[n]};
        float* to = out_of(row);
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (16 * d < D)
                *reinterpret_cast<f32x4_a4*>(to + 16 * d + 4 * g) = l[n] == 0.0f ? f32x4{0, 0, 0, 0} : a.joined ? o[n][d] : o[n][d] / l[n];
    }
}

template <class KV, int ND, int NT>
void launch_attn_tree_nt(const AttnArgs& a, hipStream_t s) {
    const int R = a.T * a.group;
    const dim3 grid(a.kv.heads * ((R + 64 * NT - 1) / (64 * NT)), a.table.seqs, a.parts);
    hipLaunchKernelGGL((k_attn_tree<KV, ND, NT>), grid, dim3(256), (TreeAttn<KV, ND, NT>::LDS), s, a);
}

template <class KV, int ND>
void launch_attn_tree_nd(const AttnArgs& a, hipStream_t s) {
    if constexpr (ND <= 8)
        if (a.tiles == 2) return launch_attn_tree_nt<KV, ND, 2>(a, s);
    launch_attn_tree_nt<KV, ND, 1>(a, s);
}

template <class KV>
void launch_attn_tree_part(const AttnArgs& a, hipStream_t s) {
    if (a.kv.dim <= 64) launch_attn_tree_nd<KV, 4>(a, s);
    else if (a.kv.dim <= 128) launch_attn_tree_nd<KV, 8>(a, s);
    else if (a.kv.dim <= 192) launch_attn_tree_nd<KV, 12>(a, s);
    else launch_attn_tree_nd<KV, 16>(a, s);
}

}  // namespace kq
