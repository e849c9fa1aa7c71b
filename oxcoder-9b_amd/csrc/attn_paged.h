// Attention over a paged key-value cache, the part that reads the cache (attn_paged.hip joins the parts).
//
//   out = sum_p e_p v_p / sum_p e_p,   e_p = 2^(x_p - m),   x_p = scale log2(e) q.k_p,   m = max x_p
//
// A request's positions fall into chunks of AT_CHUNK; a workgroup takes one, two or four chunks of one key-value head for up to
// 16 or 32 of the rows (tokens x query heads of the group) that read them.  It leaves each row's m, sum e and sum e v of each
// chunk, or of each pair of chunks; chunks and pairs lie at fixed places and are joined in the same steps wherever that
// happens, so a row's result does not depend on what else runs.  A wave takes 64 neighbouring positions in steps
// of 32, keys and values straight from memory to registers and the next step's (or the next chunk's) in flight while it
// computes, with 16x16x32 MFMAs for 16 rows at a time:
//   S^T [position][row] = K [position][d] Q^T [d][row],   O^T [d][row] += V^T [d][position] E^T [position][row].
// The result layout of the first (lane: row lane % 16, positions 4 (lane / 16) + 0..3 of a tile) is the operand layout of the
// second for an order of positions that V's loads follow, so e never leaves its lane.  V^T comes from V by byte
// permutes: a lane loads 1, 2, 4 or 8 neighbouring d of the 8 positions whose values it feeds.
//
// q and e are fp32; the cache's types multiply them exactly when they are cut into three parts of 8 (bf16) or
// 11 (f16) bits, each part truncated from what the one before left, so products are those of fp32 and the sums fp32.  What
// f16's range does not hold of an element or a weight far below the largest is made up for by fp32 products.
// Three products in place of one cost little: the kernel waits for memory.  An 8-bit cache's codes are bf16 values to q and e.
//
// Measured: 48 requests of up to 8191 positions, 32 query heads on 8 of 128 bf16 values, pages of 16 (823 MB) 145 us, 5.7 TB/s
// where a bare read of the same places reaches 6.1; matrix units busy 11 % of the time, vector units 24 %, waves wait to
// issue loads half of theirs and for data a third.  With two of three products left out, with all matrix instructions
// replaced and with no exponentials the time stays; a part for every chunk (2 KB) instead of every second one costs 9 us, more
// than its bytes explain.  32 requests of 16384 8-bit positions (572 MB): 135 us, 4.2 TB/s, vector units 56 % (a step converts 64
// codes of keys and 64 of values a lane, with 64 byte permutes; queries as 24-bit integers of their row's largest would spare the
// keys' half and measured 131, but leave a small element fewer bits).  f16, 8 drafts of 4 tokens, 16 query heads on 4 of 256
// values (92 MB): 28 us.  Joining in the last workgroup to end, with tickets, in place of a launch of its
// own measured slower everywhere (8 requests of 5003, 4 tokens: 34 -> 82 us; 48 requests: 173 -> 181 us).
#pragma once
#include <type_traits>

#include "kv_device.h"

namespace kq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int AT_CHUNK = 256;                 // positions of a chunk
constexpr int AT_WAVES = 4;

// v_perm: bytes 0..3 of the second operand are selected by 0..3, of the first by 4..7.
__device__ __forceinline__ uint32_t lo_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t hi_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Lane i's v.
__device__ __forceinline__ uint32_t of_lane(int i, uint32_t v) { return (uint32_t)__builtin_amdgcn_ds_bpermute(i << 2, (int)v); }

__device__ __forceinline__ float fbits(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t ubits(float f) { return __builtin_bit_cast(uint32_t, f); }

// Both elements' three parts of 8 bits, packed in pairs.  A part that is left with nothing becomes a number of x's sign far
// below the last part's step (0 for x = 0), so that an infinite factor gives an infinity and not 0 * inf.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    auto cut = [](float a) { return fbits(ubits(a) & 0xffff0000u); };
    // a rest that is not 0 is at least 2^-24 |x| and has at most 16 bits: the sum with 2^-50 x rounds back to it
    const float tx = x * 0x1p-50f, ty = y * 0x1p-50f;
    const float rx = x - cut(x), ry = y - cut(y), sx = rx - cut(rx), sy = ry - cut(ry);
    p0 = hi_halves(ubits(x), ubits(y));
    p1 = hi_halves(ubits(rx + tx), ubits(ry + ty));
    p2 = hi_halves(ubits(sx + tx), ubits(sy + ty));
}

// Three f16 parts of 11 bits of |x|, |y| < 2^15, x = p0 + 2^-11 p1 + 2^-22 p2: held 2^11 times larger than the one before,
// so that no rest meets f16's last step before its 24 bits are used up.  Exact from 2^-23 on, and for 0.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    auto cut = [](float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)); };
    p0 = cut(x, y);
    const float rx = (x - f16_lo(p0)) * 0x1p11f, ry = (y - f16_hi(p0)) * 0x1p11f;
    p1 = cut(rx, ry);
    p2 = cut((rx - f16_lo(p1)) * 0x1p11f, (ry - f16_hi(p1)) * 0x1p11f);
}
// What the parts leave of x.
__device__ __forceinline__ float split_rest(float x) {
#pragma unroll
    for (int i = 0; i < 3; i++) x = (x - f16_lo(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, 0.0f)))) * 0x1p11f;
    return x * 0x1p-33f;
}

template <class KV>
__device__ __forceinline__ void split2(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    if constexpr (KV::id == KQ_KV_F16) split_f16(x, y, p0, p1, p2);
    else split_bf16(x, y, p0, p1, p2);
}

template <class KV>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (KV::id == KQ_KV_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// One product of four positions, a group of 16 lanes each.
__device__ __forceinline__ f32x4 mma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Four codes (bytes of w) as floats' bits; their high halves are the codes in bf16.
__device__ __forceinline__ u32x4 code_floats(uint32_t w) {
    return u32x4{ubits((float)(int8_t)(w & 0xff)), ubits((float)(int8_t)(w >> 8 & 0xff)),
                 ubits((float)(int8_t)(w >> 16 & 0xff)), ubits((float)(int8_t)(w >> 24))};
}
// Eight codes as bf16; unpacked here, as the compiler would do it where they are loaded and hold them in four times the registers.
__device__ __forceinline__ u32x4 code_bf16(uint32_t a, uint32_t b) {
    asm volatile("" : "+v"(a), "+v"(b));
    const u32x4 x = code_floats(a), y = code_floats(b);
    return u32x4{hi_halves(x.x, x.y), hi_halves(x.z, x.w), hi_halves(y.x, y.y), hi_halves(y.z, y.w)};
}

// W neighbouring elements of V as dwords (one element: in the low half).
template <int BYTES>
struct VRaw {
    static constexpr int N = (BYTES + 3) / 4;
    uint32_t u[N];
    __device__ __forceinline__ void load(const uint8_t* p) {
        // read once, so first to leave the caches: the parts that the join reads stay (the 48 requests below 8192 positions
        // 178 -> 169 us; K's rows come in quarters and need the cache)
        if constexpr (BYTES == 16) {
            const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
            u[0] = x.x, u[1] = x.y, u[2] = x.z, u[3] = x.w;
        } else if constexpr (BYTES == 8) {
            const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
            u[0] = x.x, u[1] = x.y;
        } else if constexpr (BYTES == 4) u[0] = *reinterpret_cast<const uint32_t*>(p);
        else if constexpr (BYTES == 2) u[0] = *reinterpret_cast<const uint16_t*>(p);
        else u[0] = *p;
    }
};

// ND = dim / 16, taken in strips of 16 W values, W = 8, 4, 2 or 1 per lane.
constexpr int at_strips(int nd) { return nd / 8 + (nd >> 2 & 1) + (nd >> 1 & 1) + (nd & 1); }
constexpr int at_width(int nd, int s) {
    if (s < nd / 8) return 8;
    s -= nd / 8;
    for (int w = 4; w; w >>= 1)
        if (nd & w) {
            if (s == 0) return w;
            s--;
        }
    return 0;
}
constexpr int at_first(int nd, int s) {           // first value of strip s, in 16ths
    int n = 0;
    for (int i = 0; i < s; i++) n += at_width(nd, i);
    return n;
}

template <class KV, int ND, int NR>
struct Attn {
    static constexpr bool I8 = KV::id == KQ_KV_I8, F16 = KV::id == KQ_KV_F16;
    static constexpr int D = 16 * ND, EB = I8 ? 1 : 2;
    static constexpr int KL = I8 ? (ND + 3) / 4 : (ND + 1) / 2;  // 16-byte loads of a key by its 4 lanes
    static constexpr int PER = I8 ? 2 : 1, QS = PER * KL;        // products of a load by 8 values of each lane; their sum: q's shares
    static constexpr bool K_WHOLE = I8 ? ND % 4 == 0 : ND % 2 == 0;
    static constexpr int WIDE = D > 128 ? 128 : D, LD = WIDE == 128 ? 128 : WIDE + 4; // values of a round of the waves' join, row stride in LDS
    static constexpr float BIAS = F16 ? 14.0f : 0.0f;            // f16: e is held times 2^14
    static constexpr int VW = [] { int n = 0; for (int s = 0; s < at_strips(ND); s++) n += (at_width(ND, s) * EB + 3) / 4; return n; }();

    // Lane i of the wave: where position i of the chunk that is fetched lies in the pool, in bytes (a place that is there
    // where the position is not).
    uint32_t at_lo, at_hi;
    // The wave's 64 positions of a chunk: their first, which of them are to be read, lane i's scales.
    struct Span {
        int first;
        uint64_t there;
        float ks, vs;
    };
    const uint8_t *kb, *vb;
    u32x4 k[2][KL];                      // of position 16 t + lane % 16 of the step
    uint32_t v[2][4][VW];                // of positions 16 t + 4 (lane / 16) + i

    // page: the table's entry for the lane's position, or any other's where that is not below len.
    __device__ __forceinline__ Span open(const AttnArgs& a, int page, int kh, int first, int len, int lane) {
        Span n;
        n.first = first;
        const int p = first + lane;
        const bool ok = p < len && (unsigned)page < (unsigned)a.kv.pages;
        page = ok ? page : 0;
        const int off = ok ? p & (a.kv.page_size - 1) : 0;
        n.there = __ballot(ok);
        const int64_t at = (page * a.kv.page_stride + off * a.kv.pos_stride) * EB;
        at_lo = (uint32_t)at;
        at_hi = (uint32_t)(at >> 32);
        if constexpr (I8) {
            const int64_t e = page * a.kv.scale_page_stride + kh * a.kv.scale_head_stride + off * a.kv.scale_pos_stride;
            n.ks = a.kv.k_scale[e];
            n.vs = a.kv.v_scale[e];
        }
        return n;
    }
    // Byte offset of the wave's position i.
    __device__ __forceinline__ int64_t place(int i) const {
        return (int64_t)((uint64_t)of_lane(i, at_hi) << 32 | of_lane(i, at_lo));
    }
    // Keeps what follows from the lanes' places from being computed once for every step and held in registers.
    __device__ __forceinline__ void here() { asm volatile("" : "+v"(at_lo), "+v"(at_hi)); }
    __device__ __forceinline__ void load_k(int u, int r, int g) {
        here();
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t* row = kb + place(32 * u + 16 * t + r);
#pragma unroll
            for (int s = 0; s < KL; s++) {
                const int piece = 4 * s + g;
                if (s == KL - 1 && !K_WHOLE) {
                    constexpr int PIECES = D * EB / 16;
                    const u32x4 x = *reinterpret_cast<const u32x4*>(row + 16 * (piece < PIECES ? piece : 0));
                    k[t][s] = piece < PIECES ? x : u32x4{0, 0, 0, 0};
                } else {
                    k[t][s] = *reinterpret_cast<const u32x4*>(row + 16 * piece);
                }
            }
        }
    }
    __device__ __forceinline__ void load_v(int u, int r, int g) {
        here();
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) load_strip<0, 0>(v[t][i], vb + place(32 * u + 16 * t + 4 * g + i), r);
    }
    template <int S, int AT>
    static __device__ __forceinline__ void load_strip(uint32_t* to, const uint8_t* row, int r) {
        if constexpr (S < at_strips(ND)) {
            constexpr int W = at_width(ND, S);
            VRaw<W * EB> x;
            x.load(row + (16 * at_first(ND, S) + W * r) * EB);
#pragma unroll
            for (int j = 0; j < VRaw<W * EB>::N; j++) to[AT + j] = x.u[j];
            load_strip<S + 1, AT + VRaw<W * EB>::N>(to, row, r);
        }
    }

    // Bit 4 t + i: position 16 t + 4 g + i of step u is a hole, or not below `to`.
    static __device__ __forceinline__ uint32_t hidden(const Span& w, int u, int to, int g) {
        uint32_t bits = 0;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int at = 32 * u + 16 * t + 4 * g, n = to - w.first - at;    // n of the four are below `to`
            const uint32_t out = ~(uint32_t)(w.there >> at) | ~0u << min(max(n, 0), 4);
            bits |= (out & 15u) << (4 * t);
        }
        return bits;
    }
    __device__ __forceinline__ void clear_v(uint32_t bits) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool out = bits >> (4 * t + i) & 1u;
#pragma unroll
                for (int j = 0; j < VW; j++) v[t][i][j] = out ? 0u : v[t][i][j];
            }
    }
    // Whether a value at one of the positions is an infinity or NaN.
    __device__ __forceinline__ bool v_not_finite(uint32_t bits) const {
        if constexpr (I8) return false;                // codes; a position's scale counts only where e does
        constexpr uint32_t E = KV::id == KQ_KV_F16 ? 0x7c00u : 0x7f80u;
        bool any = false;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (bits >> (4 * t + i) & 1u)
#pragma unroll
                    for (int j = 0; j < VW; j++) any |= (v[t][i][j] & E) == E || (v[t][i][j] >> 16 & E) == E;
        return __any(any);
    }

    template <int S, int AT>
    __device__ __forceinline__ void pv_strip(const u32x4 (&p)[NR][3], f32x4 (&o)[NR][ND]) const {
        if constexpr (S < at_strips(ND)) {
            constexpr int W = at_width(ND, S), F = at_first(ND, S), NW = VRaw<W * EB>::N;
            auto raw = [&](int kk, int d) { return v[kk >> 2][kk & 3][AT + d]; };
            if constexpr (I8) {
#pragma unroll
                for (int d = 0; d < NW; d++) {
                    u32x4 x[8];
#pragma unroll
                    for (int kk = 0; kk < 8; kk++) x[kk] = code_floats(raw(kk, d));
#pragma unroll
                    for (int w = 4 * d; w < W && w < 4 * d + 4; w++) {
                        const u32x4 f = {hi_halves(x[0][w & 3], x[1][w & 3]), hi_halves(x[2][w & 3], x[3][w & 3]),
                                         hi_halves(x[4][w & 3], x[5][w & 3]), hi_halves(x[6][w & 3], x[7][w & 3])};
#pragma unroll
                        for (int n = 0; n < 3 * NR; n++) o[n % NR][F + w] = mma<KV>(f, p[n % NR][n / NR], o[n % NR][F + w]);
                    }
                }
            } else {
#pragma unroll
                for (int w = 0; w < W; w++) {
                    u32x4 f;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        f[j] = w & 1 ? hi_halves(raw(2 * j, w >> 1), raw(2 * j + 1, w >> 1))
                                     : lo_halves(raw(2 * j, w >> 1), raw(2 * j + 1, w >> 1));
#pragma unroll
                    for (int n = 0; n < 3 * NR; n++) o[n % NR][F + w] = mma<KV>(f, p[n % NR][n / NR], o[n % NR][F + w]);
                }
            }
            pv_strip<S + 1, AT + NW>(p, o);
        }
    }
    // f16: o += V^T (p0 + 2^-11 p1 + 2^-22 p2).
    template <int S, int AT>
    __device__ __forceinline__ void pv_strip_f16(const u32x4 (&p)[NR][3], f32x4 (&o)[NR][ND]) const {
        if constexpr (S < at_strips(ND)) {
            constexpr int W = at_width(ND, S), F = at_first(ND, S), NW = VRaw<W * EB>::N;
            auto raw = [&](int kk, int d) { return v[kk >> 2][kk & 3][AT + d]; };
#pragma unroll
            for (int w = 0; w < W; w++) {
                u32x4 f;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    f[j] = w & 1 ? hi_halves(raw(2 * j, w >> 1), raw(2 * j + 1, w >> 1))
                                 : lo_halves(raw(2 * j, w >> 1), raw(2 * j + 1, w >> 1));
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    f32x4 x = mma<KV>(f, p[n][1], mma<KV>(f, p[n][2], f32x4{}) * 0x1p-11f);
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = __builtin_fmaf(x[i], 0x1p-11f, o[n][F + w][i]);
                    o[n][F + w] = mma<KV>(f, p[n][0], x);
                }
            }
            pv_strip_f16<S + 1, AT + NW>(p, o);
        }
    }
    // The same in fp32: position kk's values and weights.
    template <int S, int AT>
    __device__ __forceinline__ void pv_strip_f32(const float (&e)[NR][2][4], f32x4 (&o)[NR][ND]) const {
        if constexpr (S < at_strips(ND)) {
            constexpr int W = at_width(ND, S), F = at_first(ND, S), NW = VRaw<W * EB>::N;
#pragma unroll
            for (int kk = 0; kk < 8; kk++)
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const uint32_t raw = v[kk >> 2][kk & 3][AT + (w >> 1)];
                    const float x = w & 1 ? f16_hi(raw) : f16_lo(raw);
#pragma unroll
                    for (int n = 0; n < NR; n++) o[n][F + w] = mma_f32(x, e[n][kk >> 2][kk & 3], o[n][F + w]);
                }
            pv_strip_f32<S + 1, AT + NW>(e, o);
        }
    }
    // f16 weights e 2^14: the parts hold every e >= 2^-37 exactly.  What they leave of a smaller one is added in fp32, and a
    // step with an infinite value goes that way alone, as a part may be 0 where its weight is not.  (All steps in fp32, 16 times
    // the matrix time: the 48 requests below 8192 positions 157 -> 164 us, 8 drafts of 4 tokens at 256 values 32.6 -> 36.6.)
    __device__ __forceinline__ void pv_f16(const float (&e)[NR][2][4], f32x4 (&o)[NR][ND]) const {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        f16x2 zero[4] = {};                                     // NaN once a value is not finite
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < VW; j++)
                zero[i & 3] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, v[i >> 2][i & 3][j]), f16x2{}, zero[i & 3]);
        const bool bad = __any(__builtin_bit_cast(uint32_t, zero[0] + zero[1] + (zero[2] + zero[3])) != 0);
        bool small = false;
#pragma unroll
        for (int j = 0; j < 8 * NR; j++) small |= ubits(e[j >> 3][j >> 2 & 1][j & 3]) - 1u < ubits(0x1p-23f) - 1u;
        const bool rest = __any(small);
        if (bad || rest) {
            float x[NR][2][4];
#pragma unroll
            for (int j = 0; j < 8 * NR; j++) {
                const float r = e[j >> 3][j >> 2 & 1][j & 3];
                x[j >> 3][j >> 2 & 1][j & 3] = bad ? r : split_rest(r);
            }
            pv_strip_f32<0, 0>(x, o);
        }
        if (!bad) {
            u32x4 p[NR][3];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    uint32_t p0, p1, p2;
                    split_f16(e[n][j >> 1][2 * (j & 1)], e[n][j >> 1][2 * (j & 1) + 1], p0, p1, p2);
                    p[n][0][j] = p0, p[n][1][j] = p1, p[n][2][j] = p2;
                }
            pv_strip_f16<0, 0>(p, o);
        }
    }
    // o += V^T E^T of the step, for NR tiles of rows; e[n][t][i] of position 16 t + 4 g + i, 0 where the row does not see it.
    __device__ __forceinline__ void pv(const Span& w, const float (&e)[NR][2][4], f32x4 (&o)[NR][ND], int u, int g) const {
        if constexpr (F16) return pv_f16(e, o);
        u32x4 p[NR][3];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = j >> 1, i = 2 * (j & 1);
            float sx = 1.0f, sy = 1.0f;
            if constexpr (I8) {
                const int at = 32 * u + 16 * t + 4 * g + i;
                sx = fbits(of_lane(at, ubits(w.vs))), sy = fbits(of_lane(at + 1, ubits(w.vs)));
            }
#pragma unroll
            for (int n = 0; n < NR; n++) {
                float x = e[n][t][i], y = e[n][t][i + 1];
                if constexpr (I8) {                              // a NaN stays one, a 0 takes no part
                    x = x == 0.0f ? x : x * sx;
                    y = y == 0.0f ? y : y * sy;
                }
                uint32_t p0, p1, p2;
                split_bf16(x, y, p0, p1, p2);
                p[n][0][j] = p0, p[n][1][j] = p1, p[n][2][j] = p2;
            }
        }
        pv_strip<0, 0>(p, o);
    }
};

// Where value d of row r lies in its row of LDS: rows of 128 have no gap between them, and fours change places instead.
template <int ND>
__device__ __forceinline__ int in_row(int r, int d) { return ND < 8 ? d : d ^ (r & 7) << 2; }

// The scales that bring two parts to their common maximum.
struct AtPair {
    float top, k0, k1, l;
};
__device__ __forceinline__ AtPair at_pair(AttnMl a, AttnMl b) {
    AtPair p;
    p.top = fmaxf(a.m, b.m);
    p.k0 = a.l != 0.0f ? __builtin_amdgcn_exp2f(a.m - p.top) : 0.0f;         // 0: the row saw nothing (a NaN counts)
    p.k1 = b.l != 0.0f ? __builtin_amdgcn_exp2f(b.m - p.top) : 0.0f;
    p.l = a.l * p.k0 + b.l * p.k1;
    return p;
}

// o's values in [16 FROM, 16 TO), times k, into row r of LDS; S: the strip.
template <int ND, int FROM, int TO, int S = 0>
__device__ __forceinline__ void put_o(float* row, const f32x4 (&o)[ND], float k, int r, int g) {
    if constexpr (S < at_strips(ND)) {
        constexpr int W = at_width(ND, S), F = at_first(ND, S);
        if constexpr (F >= FROM && F < TO) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 16 * (F - FROM) + (4 * g + i) * W;
                if constexpr (W >= 4) {
#pragma unroll
                    for (int w = 0; w < W; w += 4)
                        *reinterpret_cast<f32x4*>(row + in_row<ND>(r, d + w)) =
                            f32x4{o[F + w][i], o[F + w + 1][i], o[F + w + 2][i], o[F + w + 3][i]} * k;
                } else {
#pragma unroll
                    for (int w = 0; w < W; w++) row[in_row<ND>(r, d + w)] = o[F + w][i] * k;
                }
            }
        }
        put_o<ND, FROM, TO, S + 1>(row, o, k, r, g);
    }
}

// NR: tiles of 16 rows that a workgroup takes at once; PAIRED: it takes chunks by twos (apart from the other, whose way is
// shorter: one request of 611 positions 7.8 -> 7.0 us).
template <class KV, int ND, int NR, bool PAIRED>
__global__ void __launch_bounds__(64 * AT_WAVES, ND > 8 || NR > 1 ? 2 : ND > 4 ? 3 : 4) k_attn_part(AttnArgs a) {
    typedef Attn<KV, ND, NR> A;
    __shared__ u32x4 sq[NR][A::QS][3][64];                      // q's parts [tile][share][part][lane]
    __shared__ float sm[AT_WAVES][16 * NR], sl[AT_WAVES][16 * NR], st[16 * NR];
    // the first chunk of a pair: its m and l; the pair's scales
    __shared__ AttnMl held_ml[16 * NR];
    __shared__ float k0[16 * NR], k1[16 * NR];
    __shared__ int sf[AT_WAVES];
    // the waves' sums of up to 16 rows [wave][row][LD], then the first chunk's of a pair [tile][round][row, value], which only
    // the thread that put them there reads (with these as many rows as there are, so that three workgroups fit a CU)
    extern __shared__ __attribute__((aligned(16))) float sums[];
    constexpr int ROUNDS = ND > 8 ? 2 : 1;
    const int live = PAIRED ? min(16, a.T * a.group) : 16;
    auto so = [&](int w, int row) { return sums + (w * live + row) * A::LD; };
    f32x4* const held = reinterpret_cast<f32x4*>(sums + AT_WAVES * live * A::LD);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    // Workgroups go to the XCDs in turn: neighbours are heads, then requests, turned by the chunk, so that requests of
    // different lengths load the XCDs alike (chunks side by side: the 48 requests below 8192 positions took 209 us, XCD 0
    // with 1.5 times the chunks of XCD 7)
    int c = PAIRED ? 2 * blockIdx.z : blockIdx.z;
    const int group = a.row_groups > 1 ? blockIdx.x / a.kv.heads : 0, kh = blockIdx.x - group * a.kv.heads, r0 = 16 * NR * group;
    const int b = __builtin_amdgcn_readfirstlane((blockIdx.y + blockIdx.z) % gridDim.y), stride = gridDim.z;
    // every argument in one go, then the length and the table's entry side by side
    KQ_ARGS_READY("s"(a.kv.k), "s"(a.kv.v), "s"(a.kv.k_scale), "s"(a.kv.v_scale), "s"(a.kv.page_stride), "s"(a.kv.head_stride),
                  "s"(a.kv.pos_stride), "s"(a.table.pages), "s"(a.table.ld), "s"(a.lens), "s"(a.q), "s"(a.ldq));
    const int32_t* table = a.table.pages + (int64_t)b * a.table.ld;
    auto entry = [&](int first) { return table[min(first + lane, a.table.cap - 1) >> a.page_shift]; };
    const int length = a.lens[b];
    int page = entry(c * AT_CHUNK + 64 * wave);
    asm volatile("" : "+v"(page));
    const int len = min(__builtin_amdgcn_readfirstlane(length), a.max_len);
    if (c * AT_CHUNK >= len && (c || a.joined)) return;         // the join knows the chunks that are there
    const int G = a.group, R = a.T * G;
    const int all = len - a.T + 1;                              // positions that every token sees
    A s;
    s.kb = static_cast<const uint8_t*>(a.kv.k) + (int64_t)kh * a.kv.head_stride * A::EB;
    s.vb = static_cast<const uint8_t*>(a.kv.v) + (int64_t)kh * a.kv.head_stride * A::EB;
    typename A::Span w;
    bool ready = false;                                         // the chunk's first step is in flight and q's parts are there
    bool apart = false;                                         // token by token (below)
    int tok = 0;
    float f[NR], up[NR];                                        // f: what a score is multiplied by; up: what q's parts were
    bool rest = false;                                          // f16: they leave something of some element
#pragma unroll
    for (int n = 0; n < NR; n++) up[n] = 1.0f;
    for (;;) {
        // (Taken anew for each chunk, as the thread's place below: what queries' addresses come from is not held.)
        int row[NR], t[NR], lane_row = r, lane_g = g;
        asm volatile("" : "+v"(lane_row), "+v"(lane_g));
#pragma unroll
        for (int n = 0; n < NR; n++) row[n] = r0 + lane_row + 16 * n, t[n] = row[n] / G;
        typedef f32x4 Share[2];
        auto share = [&](int tile, int n, Share& x, bool again = false) {
            int at = row[tile], place = lane_g;
            if (again) asm volatile("" : "+v"(at), "+v"(place));   // read again, not held
            const float* q = a.q + ((int64_t)b * a.T + (at < R ? again ? at / G : t[tile] : 0)) * a.ldq +
                             (int64_t)(at < R ? kh * G + at % G : 0) * A::D;
            const int d = 32 * A::PER * (n / A::PER) + 8 * (A::PER * place + n % A::PER);
            const bool ok = A::K_WHOLE || n < A::QS - A::PER || d < A::D;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                x[j] = *reinterpret_cast<const f32x4_a4*>(q + (ok ? d : 0) + 4 * j);
                if (!ok) x[j] = f32x4{0, 0, 0, 0};
            }
        };
        if (!ready) {
            w = s.open(a, page, kh, c * AT_CHUNK + 64 * wave, len, lane);
            // q's parts; each wave cuts a share
            constexpr int SHARES = (A::QS + AT_WAVES - 1) / AT_WAVES, WHOLE = A::F16 ? A::QS : 0;
            Share mine[NR][SHARES], whole[NR][WHOLE ? WHOLE : 1];
#pragma unroll
            for (int tile = 0; tile < NR; tile++) {
#pragma unroll
                for (int i = 0; i < SHARES; i++) share(tile, min(AT_WAVES * i + wave, A::QS - 1), mine[tile][i]);
#pragma unroll
                for (int n = 0; n < WHOLE; n++) share(tile, n, whole[tile][n]);
            }
            s.load_k(0, r, g);
            s.load_v(0, r, g);
            bool small = false;
#pragma unroll
            for (int tile = 0; tile < NR; tile++) {
                float top = 0.0f;
                uint32_t least = ~0u;                           // of the elements that are not 0, less one
                f[tile] = a.scale;
#pragma unroll
                for (int n = 0; n < WHOLE; n++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float x = fabsf(whole[tile][n][j >> 2][j & 3]);
                        top = fmaxf(top, x);
                        least = min(least, ubits(x) - 1u);
                    }
                if constexpr (A::F16) {
                    // times a power of two that puts the row's largest near 2^14
                    top = xor32_max(xor16_max(top));
                    const uint32_t ex = max(ubits(top) >> 23, 15u);
                    up[tile] = fbits(min(268u - ex, 254u) << 23);
                    f[tile] *= fbits((ex - 14u) << 23);
                    small |= least < ((max(ex, 38u) - 37u) << 23) - 1u;   // an element below 2^-37 of the largest's power
                }
#pragma unroll
                for (int i = 0; i < SHARES; i++) {
                    const int n = AT_WAVES * i + wave;
                    if (n < A::QS) {
                        u32x4 p[3];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint32_t p0, p1, p2;
                            split2<KV>(mine[tile][i][j >> 1][2 * (j & 1)] * up[tile], mine[tile][i][j >> 1][2 * (j & 1) + 1] * up[tile], p0, p1, p2);
                            p[0][j] = p0, p[1][j] = p1, p[2][j] = p2;
                        }
#pragma unroll
                        for (int j = 0; j < 3; j++) sq[tile][n][j][16 * lane_g + lane_row] = p[j];
                    }
                }
            }
            rest = __any(small);
            __syncthreads();
        }
        // The next chunk: where there is one, every wave has both its steps in this one.
        const bool first_of_two = PAIRED && !(c & 1) && (int64_t)(c + 1) * AT_CHUNK < len;
        const int after = first_of_two ? c + 1 : PAIRED ? (c & ~1) + 2 * stride : c + stride;
        const bool on = !apart && (int64_t)after * AT_CHUNK < len;
        int page_on = -1;
        typename A::Span wn = w;
        float m[NR], l[NR];
        f32x4 o[NR][ND] = {};
#pragma unroll
        for (int n = 0; n < NR; n++) m[n] = -INFINITY, l[n] = 0.0f;
        int found = 0;
#pragma unroll 1
        for (int u = 0; u < 2; u++) {
            const int base = w.first + 32 * u;
            if (base >= len) break;
            float e[NR][2][4];
            f32x4 acc[NR][2] = {};
            if constexpr (A::F16) {
#pragma unroll
                for (int j = 2; j >= 0; j--)
#pragma unroll
                    for (int n = 0; n < A::QS; n++)
#pragma unroll
                        for (int tile = 0; tile < NR; tile++) {
                            const u32x4 qp = sq[tile][n][j][lane];
#pragma unroll
                            for (int i = 0; i < 2; i++)
                                acc[tile][i] = mma<KV>(s.k[i][n], qp, n || j == 2 ? acc[tile][i] : acc[tile][i] * 0x1p-11f);
                        }
                // S^T of q's elements, or of what the parts leave of them, in fp32.
                auto in_fp32 = [&](f32x4 (&to)[NR][2], bool left) {
#pragma unroll
                    for (int n = 0; n < A::QS; n++)
#pragma unroll
                        for (int tile = 0; tile < NR; tile++) {
                            __builtin_amdgcn_sched_barrier(0);  // (one share's registers at a time)
                            Share x;
                            share(tile, n, x, true);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                float y = x[j >> 2][j & 3] * up[tile];
                                if (left) y = split_rest(y);
#pragma unroll
                                for (int i = 0; i < 2; i++) {
                                    uint32_t raw = s.k[i][n][j >> 1];
                                    asm volatile("" : "+v"(raw));
                                    to[tile][i] = mma_f32(j & 1 ? f16_hi(raw) : f16_lo(raw), y, to[tile][i]);
                                }
                            }
                        }
                    __builtin_amdgcn_sched_barrier(0);
                };
                if (rest) in_fp32(acc, true);
                bool nan = false;                               // an infinite key, it may be, times a part that is 0
#pragma unroll
                for (int j = 0; j < 8 * NR; j += 2)
                    nan |= __builtin_isunordered(acc[j >> 3][j >> 2 & 1][j & 3], acc[j >> 3][j >> 2 & 1][(j & 3) + 1]);
                if (__any(nan)) {
                    f32x4 whole[NR][2] = {};
                    in_fp32(whole, false);
#pragma unroll
                    for (int j = 0; j < 8 * NR; j++) {
                        const float x = acc[j >> 3][j >> 2 & 1][j & 3];
                        acc[j >> 3][j >> 2 & 1][j & 3] = x == x ? x : whole[j >> 3][j >> 2 & 1][j & 3];
                    }
                }
            } else {
#pragma unroll
                for (int n = 0; n < A::QS; n++) {
                    u32x4 key[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if constexpr (A::I8) key[i] = code_bf16(s.k[i][n / 2][2 * (n & 1)], s.k[i][n / 2][2 * (n & 1) + 1]);
                        else key[i] = s.k[i][n];
                    }
#pragma unroll
                    for (int tile = 0; tile < NR; tile++) {
                        u32x4 qp[3];
#pragma unroll
                        for (int j = 0; j < 3; j++) qp[j] = sq[tile][n][j][lane];
#pragma unroll
                        for (int j = 2; j >= 0; j--)
#pragma unroll
                            for (int i = 0; i < 2; i++) acc[tile][i] = mma<KV>(key[i], qp[j], acc[tile][i]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8 * NR; j++) e[j >> 3][j >> 2 & 1][j & 3] = acc[j >> 3][j >> 2 & 1][j & 3];
            // What the next step reads is fetched whether there is one or not (no place that is not there is read, all lanes
            // take the pool's first): the waits below then know how many loads are younger than theirs.
            if (u) wn = s.open(a, on ? page_on : -1, kh, after * AT_CHUNK + 64 * wave, len, lane);
            s.load_k(1 - u, r, g);
            page_on = entry(after * AT_CHUNK + 64 * wave);
            if constexpr (A::I8) asm volatile("" : "+v"(w.ks), "+v"(w.vs));   // as here()
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float ks = 1.0f;
                if constexpr (A::I8) ks = fbits(of_lane(32 * u + 16 * (j >> 2) + 4 * g + (j & 3), ubits(w.ks)));
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    if constexpr (A::I8) e[n][j >> 2][j & 3] *= ks;
                    e[n][j >> 2][j & 3] *= f[n];
                }
            }
            // some row does not see some position
            const bool partly = (uint32_t)(w.there >> (32 * u)) != ~0u || base + 32 > all;
            if (partly) {
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    const uint32_t hid = A::hidden(w, u, row[n] < R ? all + t[n] : 0, g);
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (hid >> j & 1u) e[n][j >> 2][j & 3] = -INFINITY;
                }
                // An infinity or NaN that only some tokens see would reach the others as 0 * inf: then the rows are done
                // again, token by token, with the values that it does not see cleared.
                const uint32_t gone = A::hidden(w, u, apart ? all + tok : len, g);
                if (a.T > 1 && !apart) found |= s.v_not_finite(A::hidden(w, u, all, g) & ~gone);
                s.clear_v(gone);
            }
#pragma unroll
            for (int n = 0; n < NR; n++) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, e[n][j >> 2][j & 3]);
                top = fmaxf(m[n], xor32_max(xor16_max(top)));
                const float keep = m[n] == top ? 1.0f : __builtin_amdgcn_exp2f(m[n] - top);
                if (!__all(keep == 1.0f)) {
                    l[n] *= keep;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[n][d] *= keep;
                }
                m[n] = top;
                const float from = (top == -INFINITY ? 0.0f : top) - A::BIAS;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = __builtin_amdgcn_exp2f(e[n][j >> 2][j & 3] - from);
                    e[n][j >> 2][j & 3] = x;
                    l[n] += x;
                }
            }
            s.pv(w, e, o, u, g);
            s.load_v(1 - u, r, g);
        }
        // The waves' sums, joined: each scaled to the workgroup's maximum, then added.  (From here on the thread's place is
        // taken anew, so that no address is held through the steps.)
        int me = tid;
        asm volatile("" : "+v"(me));
        const int r = me & 15, g = me >> 4 & 3;
#pragma unroll
        for (int n = 0; n < NR; n++) {
            l[n] = xor32_sum(xor16_sum(l[n]));
            if (g == 0) sm[wave][16 * n + r] = m[n], sl[wave][16 * n + r] = l[n];
        }
        if (g == 0 && r == 0) sf[wave] = found;
        __syncthreads();
        if (a.T > 1 && !apart && (sf[0] | sf[1] | sf[2] | sf[3])) {
            apart = true;
            tok = a.T - 1;
            ready = false;
            page = entry(c * AT_CHUNK + 64 * wave);
            __syncthreads();
            continue;
        }
        // part of the group's first row
        const int64_t part0 = (((int64_t)b * a.kv.heads + kh) * R + r0) * a.parts + (PAIRED ? c >> 1 : c);
        const bool second_of_two = PAIRED && (c & 1);
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const int at = 16 * n + r;
            const float top = fmaxf(fmaxf(sm[0][at], sm[1][at]), fmaxf(sm[2][at], sm[3][at]));
            if (wave == 0 && g == 0) {
                float total = 0.0f;
#pragma unroll
                for (int i = 0; i < AT_WAVES; i++) {
                    const float li = sl[i][at];                 // 0: the wave saw nothing (a NaN counts)
                    total += li != 0.0f ? li * __builtin_amdgcn_exp2f(sm[i][at] - top) : 0.0f;
                }
                st[at] = total;
                if (a.joined && row[n] < R && (!apart || t[n] == tok)) {
                    AttnMl ml{top, total};
                    if (second_of_two) {
                        const AtPair p = at_pair(held_ml[at], ml);
                        k0[at] = p.k0, k1[at] = p.k1;
                        ml = AttnMl{p.top, p.l};
                    }
                    if (first_of_two) held_ml[at] = ml;
                    else a.pml[part0 + (int64_t)at * a.parts] = ml;
                }
            }
            const float k = l[n] != 0.0f ? __builtin_amdgcn_exp2f(m[n] - top) : 0.0f;
            auto round = [&](auto from, auto to) {
                constexpr int FROM = decltype(from)::value, TO = decltype(to)::value, Q = 4 * (TO - FROM);
                if (FROM || n) __syncthreads();                 // the round before has left LDS
                if (row[n] < R) {
                    if (l[n] != 0.0f) {
                        put_o<ND, FROM, TO>(so(wave, r), o[n], k, r, g);
                    } else {
#pragma unroll
                        for (int i = g; i < Q; i += 4) *reinterpret_cast<f32x4*>(so(wave, r) + in_row<ND>(r, 4 * i)) = f32x4{0, 0, 0, 0};
                    }
                }
                __syncthreads();
                for (int i = me; i < min(16, R - r0 - 16 * n) * Q; i += 64 * AT_WAVES) {
                    const int rr = i / Q, d = 4 * (i % Q);
                    auto of = [&](int w) { return *reinterpret_cast<const f32x4*>(so(w, rr) + in_row<ND>(rr, d)); };
                    f32x4 sum = (of(0) + of(1)) + (of(2) + of(3));
                    if (apart && (r0 + 16 * n + rr) / G != tok) continue;
                    if (a.joined) {
                        f32x4& first = held[(n * ROUNDS + FROM / 8) * 32 * live + i];
                        if (first_of_two) {
                            first = sum;
                            continue;
                        }
                        if (second_of_two) sum = first * k0[16 * n + rr] + sum * k1[16 * n + rr];
                        *reinterpret_cast<f32x4*>(a.po + (part0 + (int64_t)(16 * n + rr) * a.parts) * A::D + 16 * FROM + d) = sum;
                        continue;
                    }
                    const int tt = (r0 + 16 * n + rr) / G, hh = kh * G + (r0 + 16 * n + rr) % G;
                    const float total = st[16 * n + rr];
                    *reinterpret_cast<f32x4_a4*>(a.out + ((int64_t)b * a.T + tt) * a.ldo + (int64_t)hh * A::D + 16 * FROM + d) =
                        total == 0.0f ? f32x4{0, 0, 0, 0} : sum / total;
                }
            };
            round(std::integral_constant<int, 0>(), std::integral_constant<int, (ND < 8 ? ND : 8)>());
            if constexpr (ND > 8) round(std::integral_constant<int, 8>(), std::integral_constant<int, ND>());
        }
        // what comes next: this chunk's next token, or the next chunk
        ready = on;
        w = wn;
        if (apart && tok > 0) {
            tok--;
        } else {
            c = after;
            apart = false;
            if ((int64_t)c * AT_CHUNK >= len) return;
        }
        if (!ready) {
            page = entry(c * AT_CHUNK + 64 * wave);
            __syncthreads();                                    // q's parts and the sums have left LDS
        }
    }
}

template <class KV, int ND, int NR>
void launch_attn_part_nr(const AttnArgs& args, hipStream_t s) {
    AttnArgs a = args;
    const int R = a.T * a.group;
    a.row_groups = (R + 16 * NR - 1) / (16 * NR);
    const int live = a.paired && R < 16 ? R : 16, held = a.paired ? NR * (ND > 8 ? 2 : 1) * 512 : 0;
    const size_t lds = (size_t)live * (AT_WAVES * Attn<KV, ND, NR>::LD * 4 + held);
    const dim3 grid(a.kv.heads * a.row_groups, a.table.seqs, a.groups);
    if (a.paired) hipLaunchKernelGGL((k_attn_part<KV, ND, NR, true>), grid, dim3(64 * AT_WAVES), lds, s, a);
    else hipLaunchKernelGGL((k_attn_part<KV, ND, NR, false>), grid, dim3(64 * AT_WAVES), lds, s, a);
}

template <class KV, int ND>
void launch_attn_part_nd(const AttnArgs& a, hipStream_t s) {
    if constexpr (ND <= 8)
        if (a.T * a.group > 16) return launch_attn_part_nr<KV, ND, 2>(a, s);
    launch_attn_part_nr<KV, ND, 1>(a, s);
}

template <class KV>
void launch_attn_part(const AttnArgs& a, hipStream_t s) {
    static constexpr void (*go[16])(const AttnArgs&, hipStream_t) = {
        launch_attn_part_nd<KV, 1>, launch_attn_part_nd<KV, 2>, launch_attn_part_nd<KV, 3>, launch_attn_part_nd<KV, 4>,
        launch_attn_part_nd<KV, 5>, launch_attn_part_nd<KV, 6>, launch_attn_part_nd<KV, 7>, launch_attn_part_nd<KV, 8>,
        launch_attn_part_nd<KV, 9>, launch_attn_part_nd<KV, 10>, launch_attn_part_nd<KV, 11>, launch_attn_part_nd<KV, 12>,
        launch_attn_part_nd<KV, 13>, launch_attn_part_nd<KV, 14>, launch_attn_part_nd<KV, 15>, launch_attn_part_nd<KV, 16>};
    go[a.kv.dim / 16 - 1](a, s);
}

}  // namespace kq
