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
//
// Nearest its products where there are many rows: 64 nodes over 50001 positions, 32 on 8 heads of 128, bf16, take three times
// 52 GFLOP in 147 us, 1.07 PFLOP/s, 86 % of a large bf16 product's rate; the matrix units are busy 58 % of the clocks, and waves wait
// for their turn to issue 40 % of theirs (a kernel whose waves each read the cache for themselves, as for a few tokens a request:
// 240).  With fewer, by what is done once a tile: fetching, converting and storing it for 64 rows (16 requests of 24 nodes, 16 on
// 4 heads of 256, f16: 179 us, whose products alone would take 68; 32 of 16 nodes, 8-bit: 161, and 85).  Two tiles of rows a wave
// (NT = 2) halve that where there are more than 64 rows (the long context 148 us against 173), but heads above 128 leave no registers
// for them.  Tiles are in LDS twice where two fit in 72 KB, so that one is filled while the other is read (a barrier a tile instead of
// two).  Times of the kernel alone, from a trace.
#pragma once
#include "attn_paged.h"

namespace kq {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// What two values lose when they are cut to bf16: a dot product of the packed halves with (-1, 0) or (0, -1) and the value, whose
// sum is exact as the rest has fewer bits than the value.  (In registers that the compiler does not see through: it takes the other
// half of one of these as a literal.)
struct Cut {
    uint32_t x, y;
    __device__ __forceinline__ Cut() : x(0x0000bf80u), y(0xbf800000u) { asm volatile("" : "+s"(x), "+s"(y)); }
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    __device__ __forceinline__ float rest(uint32_t p, uint32_t which, float v) const {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), __builtin_bit_cast(bf16x2, which), v, false);
    }
    // both values' three parts, the first value in the low half
    __device__ __forceinline__ void split3(float v, float w, uint32_t& p0, uint32_t& p1, uint32_t& p2) const {
        p0 = hi_halves(ubits(v), ubits(w));
        v = rest(p0, x, v), w = rest(p0, y, w);
        p1 = hi_halves(ubits(v), ubits(w));
        v = rest(p1, x, v), w = rest(p1, y, w);
        p2 = hi_halves(ubits(v), ubits(w));
    }
    // eight f16 values as the sums of two bf16 values; of an infinity or NaN the second is NaN
    __device__ __forceinline__ void f16_pair(u32x4 raw, u32x4& hi, u32x4& lo) const {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float v = f16_lo(raw[j]), w = f16_hi(raw[j]);
            hi[j] = hi_halves(ubits(v), ubits(w));
            lo[j] = hi_halves(ubits(rest(hi[j], x, v)), ubits(rest(hi[j], y, w)));
        }
    }
};

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
    // bytes of a position in LDS: 8 keys' pieces of 16, and 4 values' pieces of 32, each fall on all banks
    static constexpr int KROW = 2 * D + 16, VROW = 2 * D + 32;
    static constexpr int KPLANE = P * KROW, VPLANE = P * VROW, VALUES = PLANES * KPLANE, TILE = VALUES + PLANES * VPLANE;
    static constexpr int NBUF = 2 * TILE <= 72 * 1024 ? 2 : 1;
    static constexpr int UNITS = D * EB / 16;              // 16-byte pieces of a position
    static constexpr int MINE = 8;                         // positions that a wave fetches
    static constexpr int PER = (MINE * UNITS + 63) / 64;   // pieces of a lane
    static constexpr size_t LDS = (size_t)TILE * NBUF;
};

template <class KV, int ND, int NT>
__global__ void __launch_bounds__(256, ND * NT <= 4 ? 4 : ND * NT <= 8 && NT == 1 ? 3 : 2) k_attn_tree(AttnArgs a) {
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
    const Cut cut;

    // what the rows see of the tree, and what any row does
    const uint64_t* seen = a.seen + (int64_t)b * a.T;
    const uint64_t word = lane < a.T ? seen[lane] : 0;
    uint32_t lo = (uint32_t)word, hi = (uint32_t)(word >> 32);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) lo |= of_lane(lane ^ i, lo), hi |= of_lane(lane ^ i, hi);
    const uint64_t some = (uint64_t)__builtin_amdgcn_readfirstlane(hi) << 32 | __builtin_amdgcn_readfirstlane(lo);
    // (Read again where it is needed, and the thread's place below taken anew for each tile: neither is held.)
    auto here = [&]() __attribute__((always_inline)) {
        uint32_t i = lane;
        asm volatile("" : "+v"(i));
        return i;
    };
    auto nodes_of = [&](int n) __attribute__((always_inline)) {
        return seen[min((row0 + 16 * n + (int)(here() & 15)) / G, a.T - 1)];
    };

    // Keys past the head's size stay 0 from here on.
    if (D < A::D)
        for (int i = tid; i < A::NBUF * A::PLANES * A::P; i += 256) {
            uint8_t* row = tiles + i / (A::PLANES * A::P) * A::TILE + i % (A::PLANES * A::P) * A::KROW;
            for (int d = D; d < A::D; d += 8) *reinterpret_cast<u32x4*>(row + 2 * d) = u32x4{0, 0, 0, 0};
        }

    // Fetching: each wave MINE positions, a lane PER pieces of 16 bytes.  (Lanes past the last piece, and pieces past the head's size,
    // take one that another lane has too.)
    const int32_t* table = a.table.pages + (int64_t)b * a.table.ld;
    const uint8_t* kb = static_cast<const uint8_t*>(a.kv.k) + (int64_t)kh * a.kv.head_stride * A::EB;
    const int64_t to_v = static_cast<const uint8_t*>(a.kv.v) - static_cast<const uint8_t*>(a.kv.k);
    const uint32_t page_bytes = (uint32_t)a.kv.page_stride * A::EB, pos_bytes = (uint32_t)a.kv.pos_stride * A::EB;   // below 2^31 both
    const uint32_t last = D * A::EB - 16;
    auto pos_of = [&](int i, uint32_t lane) __attribute__((always_inline)) { return (int)((64 * i + lane) / A::UNITS % A::MINE); };
    auto col_of = [&](int i, uint32_t lane) __attribute__((always_inline)) { return min(16 * ((64 * i + lane) % A::UNITS), last); };
    int page[A::PER];
    auto look = [&](int first) __attribute__((always_inline)) {
        const uint32_t lane = here();
#pragma unroll
        for (int i = 0; i < A::PER; i++) page[i] = table[min(first + A::MINE * wave + pos_of(i, lane), a.table.cap - 1) >> a.page_shift];
    };
    u32x4 kreg[A::PER], vreg[A::PER];
    uint64_t ok_lanes[A::PER];
    float ks[A::PER], vs[A::PER];
    bool wild = false;                                         // values that are not finite count as 0 (below)
    auto fetch = [&](int first) __attribute__((always_inline)) {
        const uint32_t lane = here();
#pragma unroll
        for (int i = 0; i < A::PER; i++) {
            const int p = first + A::MINE * wave + pos_of(i, lane), node = p - base;
            bool ok = (unsigned)page[i] < (unsigned)a.kv.pages;
            if (first + A::P > min(base, to)) ok = ok && p < to && (node < 0 || (node < 64 && (some >> (node & 63) & 1u)));
            const uint32_t pg = ok ? page[i] : 0, off = ok ? p & (a.kv.page_size - 1) : 0;
            ok_lanes[i] = __ballot(ok);
            const uint8_t* at = kb + (uint64_t)pg * page_bytes + (uint64_t)off * pos_bytes + col_of(i, lane);
            kreg[i] = *reinterpret_cast<const u32x4*>(at);
            vreg[i] = *reinterpret_cast<const u32x4*>(at + to_v);
            if constexpr (A::I8) {
                // a position's scales by the lane that has its first piece
                if ((64 * i + lane) % A::UNITS == 0) {
                    const int64_t e = pg * a.kv.scale_page_stride + kh * a.kv.scale_head_stride + off * a.kv.scale_pos_stride;
                    ks[i] = ok ? a.kv.k_scale[e] : 0.0f;
                    vs[i] = ok ? a.kv.v_scale[e] : 0.0f;
                }
            }
        }
    };
    auto put = [&](int buf) __attribute__((always_inline)) {
        const uint32_t lane = here();
        uint8_t* kt = tiles + buf * A::TILE + A::MINE * wave * A::KROW;
        uint8_t* vt = tiles + buf * A::TILE + A::VALUES + A::MINE * wave * A::VROW;
        uint32_t ok_bits = (1u << A::MINE) - 1u;
        uint64_t all = ~0ull;
#pragma unroll
        for (int i = 0; i < A::PER; i++) all &= ok_lanes[i];
        if (all != ~0ull) {                                    // positions that are not there
#pragma unroll
            for (int i = 0; i < A::PER; i++)
                if (!(ok_lanes[i] >> lane & 1u)) kreg[i] = vreg[i] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < A::MINE; p++) {
                constexpr int U = A::UNITS;
                ok_bits &= ~((uint32_t)(~ok_lanes[p * U / 64] >> (p * U % 64) & 1u) << p);
            }
        }
        if (!A::I8 && wild) {
#pragma unroll
            for (int i = 0; i < A::PER; i++) vreg[i] = finite<A::F16 ? 0x7c00u : 0x7f80u>(vreg[i]);
        }
#pragma unroll
        for (int i = 0; i < A::PER; i++) {
            const uint32_t pos = pos_of(i, lane), col = col_of(i, lane);
            uint8_t *kp = kt + pos * A::KROW + 2 / A::EB * col, *vp = vt + pos * A::VROW + 2 / A::EB * col;
            const u32x4 k = kreg[i], v = vreg[i];
            if constexpr (A::I8) {
                *reinterpret_cast<u32x4*>(kp) = code_bf16(k.x, k.y), *reinterpret_cast<u32x4*>(kp + 16) = code_bf16(k.z, k.w);
                *reinterpret_cast<u32x4*>(vp) = code_bf16(v.x, v.y), *reinterpret_cast<u32x4*>(vp + 16) = code_bf16(v.z, v.w);
                if ((64 * i + lane) % A::UNITS == 0) scales[buf][0][A::MINE * wave + pos] = ks[i], scales[buf][1][A::MINE * wave + pos] = vs[i];
            } else if constexpr (A::F16) {
                u32x4 hi, lo;
                cut.f16_pair(k, hi, lo);
                if (wild) lo = finite<0x7f80u>(lo);            // the second part of an infinity or NaN is 0
                *reinterpret_cast<u32x4*>(kp) = hi, *reinterpret_cast<u32x4*>(kp + A::KPLANE) = lo;
                cut.f16_pair(v, hi, lo);
                *reinterpret_cast<u32x4*>(vp) = hi, *reinterpret_cast<u32x4*>(vp + A::VPLANE) = lo;
            } else {
                *reinterpret_cast<u32x4*>(kp) = k;
                *reinterpret_cast<u32x4*>(vp) = v;
            }
        }
        if (lane == 0) there[buf][wave] = ok_bits;
    };
    look(from);
    fetch(from);

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
    // e's exponents count from -under (0 at first), which moves where one passes MOST; any: the lanes whose rows have seen a position.
    // Scores' sums start at `under`, but not where all that a row has seen lies more than FAR below 0: there the sum would be rounded
    // at its size, and a later, larger score lose its own bits to it.  Such a row's scores are summed from 0, and `under` comes after.
    constexpr float MOST = 8.0f, FAR = 16.0f;
    auto apart = [](float under) __attribute__((always_inline)) { return under > FAR ? under : 0.0f; };
    float under[NT], l[NT];
    uint64_t any[NT];
    f32x4 o[NT][ND];
    // Once, and once more where an infinity or NaN in the cache left a sum that is not finite: a value reached rows that do not see
    // it as 0 * inf.  Then such values count as 0, and are given to the rows that see them at the end.
    for (;;) {
        look(from + A::P);
        put(0);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++) {
            under[n] = 0.0f, l[n] = 0.0f, any[n] = 0;
#pragma unroll
            for (int d = 0; d < ND; d++) o[n][d] = f32x4{0, 0, 0, 0};
        }
        int buf = 0;
        for (int first = from; first < to; first += A::P) {
            const bool on = first + A::P < to;
            if (on) {
                fetch(first + A::P);
                look(first + 2 * A::P);
            }
            if (!idle) {
                const uint8_t* kt = tiles + buf * A::TILE;
                const uint8_t* vt = kt + A::VALUES;
                f32x4 acc[NT][2];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float x = A::I8 ? 0.0f : under[n] - apart(under[n]);
                    acc[n][0] = acc[n][1] = f32x4{x, x, x, x};
                }
                // A step of d (of f16, of the second parts, then of the first) for both 16 positions, the next one's on its way while it is
                // multiplied; the two in turn, so that no product waits for the one just before it.
                constexpr int KN = A::QS * A::PLANES;
                u32x4 k[2][2];
                auto key = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
                        k[i & 1][t] = *reinterpret_cast<const u32x4*>(kt + (16 * t + r) * A::KROW + 64 * (i / A::PLANES) + 16 * g +
                                                                      (A::PLANES - 1 - i % A::PLANES) * A::KPLANE);
                };
                key(0);
#pragma unroll
                for (int i = 0; i < KN; i++) {
                    if (i + 1 < KN) key(i + 1);
                    const bool first_part = i % A::PLANES == A::PLANES - 1;
#pragma unroll
                    for (int j = first_part ? 2 : 1; j >= 0; j--)
#pragma unroll
                        for (int n = 0; n < 2 * NT; n++)
                            acc[n >> 1][n & 1] = mma_bf16(k[i & 1][n & 1], qp[n >> 1][i / A::PLANES][j], acc[n >> 1][n & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (A::I8) {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const f32x4 x = *reinterpret_cast<const f32x4*>(&scales[buf][0][16 * t + 4 * g]);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            const float from = under[n] - apart(under[n]);
#pragma unroll
                            for (int i = 0; i < 4; i++) acc[n][t][i] = __builtin_fmaf(acc[n][t][i], x[i], from);
                        }
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
                    if (__ballot(top > MOST || under[n] > FAR) | (__ballot(top > -INFINITY) & ~any[n])) {
                        top = xor32_max(xor16_max(top));
                        // (by the tile's largest itself: what rounding `under` moves, far from 0, must not leave e above 1)
                        const float rest = apart(under[n]);
                        const bool had = any[n] >> lane & 1u, up = top + rest > (had ? MOST : -INFINITY);
                        const float by = up ? top : -rest, keep = had && up ? __builtin_amdgcn_exp2f(-(top + rest)) : 1.0f;
                        under[n] = up ? under[n] - rest - by : under[n];
                        any[n] |= __ballot(up);
                        l[n] *= keep;
#pragma unroll
                        for (int d = 0; d < ND; d++) o[n][d] *= keep;
#pragma unroll
                        for (int i = 0; i < 8; i++) acc[n][i >> 2][i & 3] -= by;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float x = __builtin_amdgcn_exp2f(acc[n][i >> 2][i & 3]);
                        acc[n][i >> 2][i & 3] = x;
                        l[n] += x;
                    }
                }
                {
                    u32x4 ep[NT][3];
                    if constexpr (A::I8) {
                        f32x4 x[2];
#pragma unroll
                        for (int t = 0; t < 2; t++) x[t] = *reinterpret_cast<const f32x4*>(&scales[buf][1][16 * t + 4 * g]);
                        auto scaled = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
                            for (int i = 0; i < 8 * NT; i++) {
                                const float e = acc[i >> 3][i >> 2 & 1][i & 3], y = e * x[i >> 2 & 1][i & 3];
                                acc[i >> 3][i >> 2 & 1][i & 3] = decltype(careful)::value && e == 0.0f ? e : y;
                            }
                        };
                        if (partly) scaled(std::true_type());      // a position that a row does not see takes no part, whatever its scale
                        else scaled(std::false_type());
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float e0 = acc[n][j >> 1][2 * (j & 1)], e1 = acc[n][j >> 1][2 * (j & 1) + 1];
                            uint32_t q0, q1, q2;
                            cut.split3(e0, e1, q0, q1, q2);
                            ep[n][0][j] = q0, ep[n][1][j] = q1, ep[n][2][j] = q2;
                        }
                    // four positions' values at a time, transposed: lane r's d, positions 4 g + 0..3 of each 16
                    const uint8_t* at = vt + (4 * g + (r >> 2)) * A::VROW + 8 * (r & 3);
                    constexpr int VN = ND / 2 * A::PLANES;
                    u32x4 v[2][2];
                    auto value = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                        for (int w = 0; w < 2; w++) {
                            const uint8_t* from = at + 64 * (i / A::PLANES) + 32 * w + (A::PLANES - 1 - i % A::PLANES) * A::VPLANE;
                            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)from));
                            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(from + 16 * A::VROW)));
                            v[i & 1][w] = u32x4{x.x, x.y, y.x, y.y};
                        }
                    };
                    value(0);
#pragma unroll
                    for (int i = 0; i < VN; i++) {
                        if (i + 1 < VN) value(i + 1);
                        const bool first_part = i % A::PLANES == A::PLANES - 1;
#pragma unroll
                        for (int j = first_part ? 2 : 1; j >= 0; j--)
#pragma unroll
                            for (int n = 0; n < 2 * NT; n++) {
                                f32x4& to = o[n >> 1][2 * (i / A::PLANES) + (n & 1)];
                                to = mma_bf16(v[i & 1][n & 1], ep[n >> 1][j], to);
                            }
                        __builtin_amdgcn_sched_barrier(0);
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
        look(from);
        fetch(from);
    }
    const int me = here(), row_of_me = me & 15, d_of_me = 4 * (me >> 4);
    if (!A::I8 && wild && !idle) {
        uint64_t nodes[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) nodes[n] = nodes_of(n);
        for (int p = from; p < to; p++) {
            const int page = __builtin_amdgcn_readfirstlane(table[p >> a.page_shift]);
            if ((unsigned)page >= (unsigned)a.kv.pages) continue;
            const uint8_t* at = kb + to_v + (uint64_t)page * page_bytes + (uint64_t)(p & (a.kv.page_size - 1)) * pos_bytes + 2 * d_of_me;
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
#pragma unroll
    for (int n = 0; n < NT; n++) {
        l[n] = xor32_sum(xor16_sum(l[n]));
        if (!nodes_of(n)) l[n] = 0.0f;                           // no node: it has seen nothing
    }
    const int64_t part0 = (((int64_t)b * a.kv.heads + kh) * R) * a.parts + z;
    auto out_of = [&](int row) {
        return a.joined ? a.po + (part0 + (int64_t)row * a.parts) * D
                        : a.out + ((int64_t)b * a.T + row / G) * a.ldo + (int64_t)(kh * G + row % G) * D;
    };
    if (idle) return;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int row = row0 + 16 * n + row_of_me;
        if (row >= R) continue;
        if (a.joined && d_of_me == 0) a.pml[part0 + (int64_t)row * a.parts] = AttnMl{l[n] != 0.0f ? -under[n] : -INFINITY, l[n]};
        float* to = out_of(row);
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (16 * d < D)
                *reinterpret_cast<f32x4_a4*>(to + 16 * d + d_of_me) = l[n] == 0.0f ? f32x4{0, 0, 0, 0} : a.joined ? o[n][d] : o[n][d] / l[n];
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
