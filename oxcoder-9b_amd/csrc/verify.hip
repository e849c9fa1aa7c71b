// Verification of drafted tokens against the target's probabilities, from given random numbers (include/kq.h: kq_verify).
//
// With p the softmax of a node's row and q the probabilities that its children were drawn from, refusing a child leaves
// max(p - q, 0) normalised, refusing another max of that less q, and so on: after k refusals max(p - a q, 0) / Z with
// a_0 = 0, Z_0 = 1, a_k+1 = a_k + Z_k, Z_k+1 = sum max(p - a_k+1 q, 0).  So what is left is one number a and the row.  For a
// child that was not drawn (q holds it alone) what is left is p without the refused tokens.
//
// A round is two kernels: the first takes softmax statistics, slice by slice, of the row that a request's walk stands at and of as
// many levels of nodes below it as fit its share of rows; the second, one workgroup a request, walks on over those and, where
// the walk ends, draws the next token: over the slices' sums, then inside one slice.  Rows that no walk comes to need not be
// read: a batch of large trees takes four rounds, the last of which reads whatever is left below the few walks that still go on.
// Where a draft's probabilities leave something else than p, two more kernels sum what is left slice by slice and draw.  The second goes on
// alone from there, a workgroup a request: a chain's refused draft ends its walk, but every further sibling that is refused, and every node
// behind one that is taken, are passes over a whole row (16 requests of 16 nodes over 151936 ids, drawn: chains 84 us, trees 569, of
// which that kernel takes 557).
//
// The statistics are bound by 64-bit arithmetic beside the loads (155 MB, 39 million weights: 47 us, 3.3 TB/s; 70 with a polynomial of
// degree 11, one weight after another), the walks by latency: 4 us where nothing is drawn, 12 with a draw (its two scans), for a
// whole batch at once.  One request of 5 nodes over 151936 ids: 19 us; 32 chains of 8 with draft probabilities: 87; 16 trees of
// 64 nodes over 248320 ids: 90, where a copy's rate would take 200 for all 1 GB of their rows.
#include <algorithm>

#include "kq_device.h"
#include "kq_internal.h"

namespace kq {

constexpr int VF_T = 256;                    // threads of the kernels that read rows
constexpr int VF_MOST = 4096;                // ids of their slices
constexpr int VF_LEAST = 2048;               // or half of that
constexpr int VF_W = 1024;                   // threads of the walk
constexpr int VF_EACH = VF_MOST / VF_W;      // ids of one of them in a slice
constexpr int VF_ROUNDS = 4;

// Weights are held in 64 bits as well: a vocabulary's running sum has a border for every id, and fp32 weights, off by 2^-24
// each, would put one draw in some hundred on the border's other side.
struct VfScale {
    double c, least;           // log2(e) / temperature; a difference of logits whose weight is 0
    bool greedy;               // temperature 0: the first of the largest logits alone
};
__device__ __forceinline__ VfScale vf_scale(const VerifyArgs& a, int b) {
    const float t = a.temperature ? a.temperature[b] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const double x = greedy ? 1.0 : fmin((double)t, 3e38);
    return VfScale{1.4426950408889634 / x, -1400.0 * x, greedy};
}
// 2^f of f in -1/2..1/2 to within 2e-14 of it: the polynomial of degree 9 that equals it at Chebyshev's points, the highest power first.
constexpr int VF_TERMS = 10;
__device__ constexpr double VF_POLY[VF_TERMS] = {
    1.0205905413765595e-07, 1.325964524488711e-06, 1.5252672924850737e-05, 0.0001540343375125101,
    0.0013333558200794592, 0.009618129193934313, 0.05550410866465167, 0.2402265069564034,
    0.6931471805599462, 1.0000000000000135};
// For a loop of them: in scalar registers (as literals the compiler copies one for each step).
struct VfPoly {
    double c[VF_TERMS];
    __device__ __forceinline__ VfPoly() {
#pragma unroll
        for (int k = 0; k < VF_TERMS; k++) {
            c[k] = VF_POLY[k];
            asm volatile("" : "+s"(c[k]));
        }
    }
};
// x's weight beside the row's largest logit m, 2^(c (x - m)): 0 for -inf and NaN; beside +inf, 1 for that alone.  To within 4e-14 of
// it.  (c x - c m would be off by the rounding of c m, which a low temperature makes large.)
struct VfTop {
    float m;
    double c, least;
    __device__ __forceinline__ VfTop(const VfScale& s, float top) : m(top), c(s.c), least(s.least) {}
    // N of them side by side, as a 64-bit instruction's result comes late
    template <int N>
    __device__ __forceinline__ void weights(const double (&poly)[VF_TERMS], const float (&x)[N], double (&w)[N]) const {
        if (m == INFINITY) {
#pragma unroll
            for (int i = 0; i < N; i++) w[i] = x[i] == m ? 1.0 : 0.0;
            return;
        }
        double f[N], t[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const double z = fmax((double)x[i] - (double)m, least) * c;
            t[i] = z + 0x1.8p52;                               // its low half is z to the nearest integer
            f[i] = z - (t[i] - 0x1.8p52);
            w[i] = poly[0];
        }
#pragma unroll
        for (int k = 1; k < VF_TERMS; k++)
#pragma unroll
            for (int i = 0; i < N; i++) w[i] = fma(w[i], f[i], poly[k]);
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = ldexp(w[i], (int)__builtin_bit_cast(uint64_t, t[i]));
    }
    __device__ __forceinline__ double weight(float x) const {
        const float one[1] = {x};
        double w[1];
        weights(VF_POLY, one, w);
        return w[0];
    }
};
__device__ __forceinline__ double vf_weight(const VfScale& s, float x, float m) { return VfTop(s, m).weight(x); }

__device__ __forceinline__ double vf_wave_sum(double v) {
#pragma unroll 1
    for (int w = 32; w; w >>= 1) v += __shfl_xor(v, w, 64);
    return v;
}

// Where a request's walk stands.
enum { VF_WALKING, VF_DONE, VF_LEFT };       // VF_LEFT: a draft was refused, and what that leaves is still to be summed
struct VfState {
    int cur, n, status, child; // the node, accepted drafts, the child that was refused
    int first;                 // the row's largest logit: its place
    float m;                   // and it
    double per;                // 1 / the sum of the row's weights
};
__device__ __forceinline__ VfState* vf_state(const VerifyArgs& a, int b) { return reinterpret_cast<VfState*>(a.ws) + b; }
__device__ __forceinline__ VerifyPart* vf_parts(const VerifyArgs& a, int64_t row) {
    return reinterpret_cast<VerifyPart*>(a.ws + a.parts_at) + row * a.slices;
}
__device__ __forceinline__ double* vf_sums(const VerifyArgs& a, int b) {
    return reinterpret_cast<double*>(a.ws + a.sums_at) + (int64_t)b * a.slices;
}

// The nodes whose rows a round looks at, by a whole wave with up = the lane's node's parent (-2: none): cur, and as many whole levels
// below it as leave at most `most` nodes.
__device__ __forceinline__ uint64_t vf_round(int up, int cur, int most) {
    const int lane = threadIdx.x & 63;
    // steps up to cur, by doubling; far: not below cur
    int link = up, steps = 1;
    bool there = lane == cur;
    if (there) link = lane, steps = 0;
#pragma unroll 1
    for (int i = 0; i < 6; i++) {
        const int from = max(link, 0);
        const int on = __shfl(link, from, 64), more = __shfl(steps, from, 64);
        if (link >= 0 && !there) {
            steps += more;
            link = on;
        }
    }
    const bool below = link == cur;
    uint64_t nodes = 1ull << cur;
#pragma unroll 1
    for (int level = 1; level < TREE_MOST; level++) {
        const uint64_t more = __ballot(below && steps <= level);
        if (more == nodes || __popcll(more) > most) break;
        nodes = more;
    }
    return nodes;
}
// The lane's node's parent, -2 where it is none.
__device__ __forceinline__ int vf_up(const VerifyArgs& a, int b, int t) {
    const int up = t < a.T ? a.parents[(int64_t)b * a.ldp + t] : -2;
    return t ? (up >= 0 && up < t ? up : -2) : up;
}

// A slice's nv values into LDS; returns the thread's largest.  (Here and below, loops that take an exponential each are kept rolled and
// code is shared where it can be: a kernel of some microseconds waits for its own instructions, some tenths of one for each KB.)
template <bool V4, int SLICE>
__device__ __forceinline__ float vf_stage(const float* x, int nv, float* to) {
    constexpr int QUADS = SLICE / VF_T / 4;
    float m = -INFINITY;
    if (nv == SLICE) {
        f32x4 v[QUADS];
#pragma unroll
        for (int n = 0; n < QUADS; n++) {
            const float* at = x + 4 * (n * VF_T + threadIdx.x);
            if constexpr (V4) v[n] = *reinterpret_cast<const f32x4*>(at);
            else v[n] = *reinterpret_cast<const f32x4_a4*>(at);
        }
#pragma unroll
        for (int n = 0; n < QUADS; n++) {
            m = fmaxf(m, fmaxf(fmaxf(v[n].x, v[n].y), fmaxf(v[n].z, v[n].w)));
            *reinterpret_cast<f32x4*>(to + 4 * (n * VF_T + threadIdx.x)) = v[n];
        }
    } else {
#pragma unroll 1
        for (int i = threadIdx.x; i < nv; i += VF_T) {
            const float v = x[i];
            to[i] = v;
            m = fmaxf(m, v);
        }
        if ((int)threadIdx.x < (-nv & 3)) to[nv + threadIdx.x] = -INFINITY;    // whole quads
    }
    return m;
}

template <bool V4, int SLICE>
__global__ void __launch_bounds__(VF_T) k_verify_stats(VerifyArgs a, int round, int most) {
    extern __shared__ __attribute__((aligned(16))) float vf_lds[];
    __shared__ float sm[VF_T / 64];
    __shared__ double ss[VF_T / 64];
    __shared__ int sa[VF_T / 64];
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int up = vf_up(a, b, lane);
    int cur = 0;
    if (round) {
        const VfState* state = vf_state(a, b);
        if (state->status != VF_WALKING) return;
        cur = state->cur;
    } else if (__shfl(up, 0, 64) != -1) {
        return;
    }
    uint64_t nodes = vf_round(up, cur, most);
    const int v0 = blockIdx.x * SLICE, nv = min(SLICE, a.V - v0);
    const VfScale s = vf_scale(a, b);
#pragma unroll 1
    for (int k = 0; nodes; nodes &= nodes - 1, k++) {
        if (k % (int)gridDim.z != (int)blockIdx.z) continue;
        const int64_t row = (int64_t)b * a.T + __builtin_ctzll(nodes);
        const float* x = a.x + row * a.ldx + v0;
        float m = vf_stage<V4, SLICE>(x, nv, vf_lds);
        for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
        __syncthreads();
        if (lane == 0) sm[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
        double sum = 0.0;
        int at = INT_MAX;
        if (m > -INFINITY) {
            const VfTop top(s, m);
            if (s.greedy) {                                    // its place alone counts
                for (int i = tid; i < nv && at == INT_MAX; i += VF_T)
                    if (vf_lds[i] == m) at = i;
            } else {
                const VfPoly poly;
#pragma unroll 1
                for (int i = 4 * tid; i < nv; i += 4 * VF_T) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(vf_lds + i);
                    const float x[4] = {v.x, v.y, v.z, v.w};
                    double w[4];
                    top.weights(poly.c, x, w);
                    sum += (w[0] + w[1]) + (w[2] + w[3]);
                }
            }
        }
        sum = vf_wave_sum(sum);
        for (int w = 32; w; w >>= 1) at = min(at, __shfl_xor(at, w, 64));
        if (lane == 0) ss[wave] = sum, sa[wave] = at;
        __syncthreads();
        if (tid == 0) {
            at = min(min(sa[0], sa[1]), min(sa[2], sa[3]));
            vf_parts(a, row)[blockIdx.x] = VerifyPart{(ss[0] + ss[1]) + (ss[2] + ss[3]), m, s.greedy && m > -INFINITY ? v0 + at : 0};
        }
    }
}

// A row's distribution as the walk left it: weights of p, less the refused tokens or a times q's.
struct VfLeft {
    const float *x, *q;        // the row; q's, or NULL
    float m;
    int first;                 // greedy: the one id that has a weight
    double a, per;             // per: 1 / sum of the weights
    int gone;                  // refused tokens, in LDS
};

struct VfShared {
    int tok[TREE_MOST], up[TREE_MOST], top_at[TREE_MOST], refused[TREE_MOST];
    float m[TREE_MOST], u[TREE_MOST], x[TREE_MOST], q[TREE_MOST];
    double sum[TREE_MOST], e[TREE_MOST], gone[TREE_MOST];     // the drafts' weights, the refused tokens'
    double wave[VF_W / 64];
    int found, last;
};

__device__ __forceinline__ double vf_left(const VfShared& S, const VfScale& s, const VfLeft& f, int i, float x, float q) {
    const double e = s.greedy ? (i == f.first ? 1.0 : 0.0) : vf_weight(s, x, f.m);
    if (f.q) return fmax(e * f.per - f.a * (double)q, 0.0);
    for (int k = 0; k < f.gone; k++)
        if (S.refused[k] == i) return 0.0;
    return e;
}

__device__ __forceinline__ double vf_left(const VfShared& S, const VfScale& s, const VfLeft& f, int i) {
    return vf_left(S, s, f, i, f.x[i], f.q ? f.q[i] : 0.0f);
}

// Sum of weight(i) over [0, n), by the whole workgroup.
template <class F>
__device__ double vf_sum(VfShared& S, F weight, int n) {
    double sum = 0.0;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += VF_W) sum += weight(i);
    sum = vf_wave_sum(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
    for (int k = 0; k < VF_W / 64; k++) sum += S.wave[k];
    return sum;
}

// The token that follows: the smallest id at which the running sum of what is left exceeds its share of the total, by the
// whole workgroup.  First over the slices, whose sums come from their statistics, or from `sums`; then inside one.  Where
// there are no sums of the slices (`rows`), and where the slice found has none left (what rounding left of refused tokens
// was its sum), over the row itself: its total, and then the id.
__device__ int vf_draw(VfShared& S, const VerifyArgs& a, const VfScale& s, const VfLeft& f, double left, const VerifyPart* parts,
                       const double* sums, bool rows) {
    extern __shared__ __attribute__((aligned(16))) double vf_w[];      // VF_MOST weights, then as many floats of q where there is one
    float* const vf_q = reinterpret_cast<float*>(vf_w + VF_MOST);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const VfTop top(s, f.m);
    double target = (double)S.u[0] * left, before = 0.0;
    int from = 0, to = a.slices, gone = f.gone;
    enum { SLICES, IDS, TOTAL, FIND };
    int found = -1;
#pragma unroll 1
    for (int what = rows ? TOTAL : SLICES; what <= FIND; what++) {
        if (what >= TOTAL) from = 0, to = a.V, before = 0.0;
        if (what == TOTAL) target = INFINITY;
        int last = -1;
        __syncthreads();
        if (tid == 0) S.found = INT_MAX, S.last = -1;
#pragma unroll 1
        for (int i0 = from; i0 < to; i0 += VF_MOST) {
            const int n = min(to - i0, VF_MOST);
            if (what != SLICES) {
                float x[VF_EACH];
#pragma unroll
                for (int k = 0; k < VF_EACH; k++) x[k] = f.x[i0 + min(k * VF_W + tid, n - 1)];
#pragma unroll
                for (int k = 0; k < VF_EACH; k++) vf_w[k * VF_W + tid] = (double)x[k];
                if (f.q) {
#pragma unroll
                    for (int k = 0; k < VF_EACH; k++) x[k] = f.q[i0 + min(k * VF_W + tid, n - 1)];
#pragma unroll
                    for (int k = 0; k < VF_EACH; k++) vf_q[k * VF_W + tid] = x[k];
                }
            }
#pragma unroll 1
            for (int i = tid; i < n; i += VF_W) {
                const int at = i0 + i, mine = what == SLICES ? a.shift : 0;
                float x = 0.0f;
                double times = 1.0;
                if (what != SLICES) x = (float)vf_w[i];
                else if (sums) times = sums[at];
                else x = parts[at].m, times = parts[at].sum;
                double w = s.greedy ? (at == f.first >> mine ? 1.0 : 0.0) : top.weight(x) * times;
                if (what == SLICES) {
                    if (sums) w = times;
                } else if (f.q) {
                    w = fmax(w * f.per - f.a * (double)vf_q[i], 0.0);
                }
                for (int k = 0; k < gone; k++)
                    if (S.refused[k] >> mine == at) w -= S.gone[k];
                vf_w[i] = w;
            }
            __syncthreads();
            // VF_EACH neighbours a thread
            const int mine = tid * VF_EACH, end = min(mine + VF_EACH, n);
            double sum = 0.0;
#pragma unroll 1
            for (int i = mine; i < end; i++) {
                sum += vf_w[i];
                if (vf_w[i] > 0.0) last = i0 + i;
            }
            double run = sum;
#pragma unroll 1
            for (int k = 1; k < 64; k <<= 1) {
                const double y = __shfl_up(run, k, 64);
                if (lane >= k) run += y;
            }
            if (lane == 63) S.wave[wave] = run;
            __syncthreads();
            double ahead = before;
#pragma unroll
            for (int k = 0; k < VF_W / 64; k++) {
                const double x = S.wave[k];
                ahead += k < wave ? x : 0.0;
                before += x;
            }
            ahead += run - sum;
            // (one lane a wave: a hundred lanes' minimum of one word takes microseconds)
            const uint64_t past = __ballot(last >= i0 + mine && ahead + sum > target);
            if (past && lane == 0) atomicMin(&S.found, 64 * wave + __builtin_ctzll(past));
            __syncthreads();
            const int who = S.found;
            if (who != INT_MAX) {
                __syncthreads();
                if (tid == who) {
                    int at = last;
#pragma unroll 1
                    for (int i = mine; i0 + i < last; i++) {
                        if (vf_w[i] > 0.0 && ahead + vf_w[i] > target) {
                            at = i0 + i;
                            break;
                        }
                        ahead += vf_w[i];
                    }
                    S.last = at, S.wave[0] = ahead;
                }
                break;
            }
        }
        const bool passed = S.found != INT_MAX;
        if (!passed && last >= 0) atomicMax(&S.last, last);    // the last with a weight: the sums' own rounding
        __syncthreads();
        found = S.last;
        if (what == SLICES) {
            if (found < 0) {
                what = IDS;
                continue;
            }
            from = found << a.shift, to = min(from + a.slice, a.V);
            before = passed ? S.wave[0] : 0.0;
            if (!passed) target = INFINITY;
        } else if (what == IDS) {
            if (found >= 0) break;
        } else if (what == TOTAL) {
            if (found < 0 && !gone) break;
            if (found < 0) gone = 0, what = IDS;               // nothing but refused tokens: `left` was rounding, the total anew from p itself
            else target = (double)S.u[0] * before;
        }
    }
    return found;
}

// The request's drafts, their logits and probabilities: a thread's, and all of them in LDS.
struct VfDraft {
    int up, tok;
    float u, x, q;
};
__device__ __forceinline__ VfDraft vf_draft(const VerifyArgs& a, int b) {
    const int t = min((int)threadIdx.x, a.T - 1);
    const int up = vf_up(a, b, t), tok = a.tokens[(int64_t)b * a.ldt + t];
    const bool in = t && up >= 0 && tok >= 0 && tok < a.V;
    const int64_t row = (int64_t)b * a.T + max(up, 0);
    const int at = in ? tok : 0;
    const float u = a.uniform[(int64_t)b * a.ldu + t], x = a.x[row * a.ldx + at], q = a.draft ? a.draft[row * a.ldd + at] : 0.0f;
    return VfDraft{up, in ? tok : -1, u, in ? x : -INFINITY, in ? q : 0.0f};
}
__device__ __forceinline__ void vf_put(VfShared& S, const VerifyArgs& a, const VfDraft& d) {
    const int t = threadIdx.x;
    if (t < a.T) S.tok[t] = d.tok, S.up[t] = d.up, S.u[t] = d.u, S.x[t] = d.x, S.q[t] = d.q;
}

// A row's statistics from its slices' by one wave: brought to the row's largest logit.
__device__ void vf_row(VfShared& S, const VerifyArgs& a, const VfScale& s, int b, int t) {
    const int lane = threadIdx.x & 63;
    const VerifyPart* p = vf_parts(a, (int64_t)b * a.T + t);
    float m = -INFINITY;
    for (int i = lane; i < a.slices; i += 64) m = fmaxf(m, p[i].m);
    for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
    double sum = 0.0;
    int at = INT_MAX;
    const VfTop top(s, m);
#pragma unroll 1
    for (int i = lane; i < a.slices; i += 64) {
        const VerifyPart y = p[i];
        if (y.m == m) at = min(at, y.at);
        sum += y.sum * top.weight(y.m);
    }
    sum = vf_wave_sum(sum);
    for (int w = 32; w; w >>= 1) at = min(at, __shfl_xor(at, w, 64));
    if (lane == 0) S.m[t] = m, S.sum[t] = m == -INFINITY ? 0.0 : s.greedy ? 1.0 : sum, S.top_at[t] = at;
}
// The same from the row itself, by the whole workgroup: a sum in another order, equal to the slices' up to 64-bit rounding.
__device__ void vf_row_anew(VfShared& S, const VerifyArgs& a, const VfScale& s, int b, int t) {
    const float* x = a.x + ((int64_t)b * a.T + t) * a.ldx;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < a.V; i += VF_W) m = fmaxf(m, x[i]);
    for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave[threadIdx.x >> 6] = (double)m;
    if (threadIdx.x == 0) S.found = INT_MAX;
    __syncthreads();
    for (int k = 0; k < VF_W / 64; k++) m = fmaxf(m, (float)S.wave[k]);
    int at = INT_MAX;
    for (int i = threadIdx.x; i < a.V; i += VF_W)
        if (x[i] == m) at = min(at, i);
    if (at != INT_MAX) atomicMin(&S.found, at);
    const double sum = m == -INFINITY ? 0.0 : vf_sum(S, [&](int i) { return vf_weight(s, x[i], m); }, a.V);
    __syncthreads();
    if (threadIdx.x == 0) S.m[t] = m, S.sum[t] = m == -INFINITY ? 0.0 : s.greedy ? 1.0 : sum, S.top_at[t] = S.found;
    __syncthreads();
}

__device__ __forceinline__ VfLeft vf_at(const VfShared& S, const VerifyArgs& a, int b, int cur) {
    return VfLeft{a.x + ((int64_t)b * a.T + cur) * a.ldx, nullptr, S.m[cur], S.top_at[cur], 0.0, 1.0 / S.sum[cur], 0};
}
__device__ __forceinline__ double vf_child(const VfShared& S, const VfScale& s, const VfLeft& f, int c) {
    return s.greedy ? (S.tok[c] == f.first ? 1.0 : 0.0) : vf_weight(s, S.x[c], f.m);
}
// cur's children with a token, those behind `past`.
__device__ __forceinline__ uint64_t vf_children(const VfShared& S, int T, int cur, int past) {
    const int t = threadIdx.x & 63;
    return __ballot(t < T && t > past && S.up[min(t, T - 1)] == cur && S.tok[min(t, T - 1)] >= 0);
}

// Walks on while the node's row has been looked at; what it says goes to the outputs, or to the state for the next round.
__global__ void __launch_bounds__(VF_W) k_verify_walk(VerifyArgs a, int round, int most) {
    __shared__ VfShared S;
    const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, T = a.T;
    VfState* const state = vf_state(a, b);
    int cur = 0, n = 0;
    if (round) {
        if (state->status != VF_WALKING) return;
        cur = state->cur, n = state->n;
    }
    const VfScale s = vf_scale(a, b);
    const VfDraft mine = vf_draft(a, b);
    const uint64_t nodes = vf_round(vf_up(a, b, tid & 63), cur, most);
    vf_put(S, a, mine);
    if (!round && a.parents[(int64_t)b * a.ldp] != -1) {       // the request sits out
        if (tid < T) a.path[(int64_t)b * T + tid] = -1;
        if (tid == 0) a.accepted[b] = a.token[b] = -1, state->status = VF_DONE;
        return;
    }
    for (int t = wave; t < T; t += VF_W / 64)
        if (nodes >> t & 1u) vf_row(S, a, s, b, t);
    __syncthreads();
    // every child's weight in its parent's row
    if (tid < T && S.up[tid] >= 0 && nodes >> S.up[tid] & 1u) {
        const int up = S.up[tid];
        S.e[tid] = s.greedy ? (S.tok[tid] == S.top_at[up] ? 1.0 : 0.0) : vf_weight(s, S.x[tid], S.m[up]);
    }
    __syncthreads();
    int* path = a.path + (int64_t)b * T;
    if (!round && tid == 0) path[0] = 0;
    for (;;) {
        VfLeft f = vf_at(S, a, b, cur);
        double left = S.sum[cur];
        int next = -1, refused = -1;
        if (left > 0.0) {
            uint64_t children = vf_children(S, T, cur, 0);
            for (; children; children &= children - 1) {
                const int c = __builtin_ctzll(children), tok = S.tok[c];
                const double e = S.e[c], u = (double)S.u[c];
                if (a.draft) {
                    if (u * (double)S.q[c] < e * f.per) next = c;
                    else refused = c;
                    break;
                }
                bool again = false;                            // refused already: it holds nothing any more
                for (int k = 0; k < f.gone; k++) again |= S.refused[k] == tok;
                const double w = again ? 0.0 : e;
                if (u * left < w) {
                    next = c;
                    break;
                }
                left -= w;
                if (!again) {
                    __syncthreads();
                    if (tid == 0) S.refused[f.gone] = tok, S.gone[f.gone] = w;
                    __syncthreads();
                    f.gone++;
                }
            }
        }
        if (next >= 0) {
            cur = next;
            n++;
            if (tid == 0) path[n] = next;
            if (nodes >> cur & 1u) {
                __syncthreads();
                continue;
            }
            if (tid == 0) state->cur = cur, state->n = n, state->status = VF_WALKING;
            return;
        }
        if (refused >= 0) {
            if (tid == 0) *state = VfState{cur, n, VF_LEFT, refused, f.first, f.m, f.per};
            return;
        }
        int token = -1;
        if (S.sum[cur] > 0.0) {
            if (!(left > 0.0)) left = S.sum[cur], f.gone = 0;  // nothing is left: drawn from p itself
            token = vf_draw(S, a, s, f, left, vf_parts(a, (int64_t)b * T + cur), nullptr, false);
        }
        for (int i = n + 1 + tid; i < T; i += VF_W) path[i] = -1;
        if (tid == 0) a.accepted[b] = n, a.token[b] = token, state->status = VF_DONE;
        return;
    }
}

// Sums over slices of max(p - q, 0) for the requests whose draft was refused.
template <bool V4, int SLICE>
__global__ void __launch_bounds__(VF_T) k_verify_left(VerifyArgs a) {
    extern __shared__ __attribute__((aligned(16))) float vf_lds[];
    __shared__ double ss[VF_T / 64];
    const int b = blockIdx.y, tid = threadIdx.x;
    const VfState state = *vf_state(a, b);
    if (state.status != VF_LEFT) return;
    const int64_t row = (int64_t)b * a.T + state.cur;
    const int v0 = blockIdx.x * SLICE, nv = min(SLICE, a.V - v0);
    const VfScale s = vf_scale(a, b);
    vf_stage<V4, SLICE>(a.x + row * a.ldx + v0, nv, vf_lds);
    vf_stage<V4, SLICE>(a.draft + row * a.ldd + v0, nv, vf_lds + SLICE);
    double sum = 0.0;
    __syncthreads();
    const VfTop top(s, state.m);
    const VfPoly poly;
#pragma unroll 1
    for (int i = 4 * tid; i < nv; i += 4 * VF_T) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(vf_lds + i), q = *reinterpret_cast<const f32x4*>(vf_lds + SLICE + i);
        const float x[4] = {v.x, v.y, v.z, v.w};
        double left[4];
        top.weights(poly.c, x, left);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double e = s.greedy ? (v0 + i + k == state.first ? 1.0 : 0.0) : left[k];
            left[k] = i + k < nv ? fmax(e * state.per - (double)q[k], 0.0) : 0.0;
        }
        sum += (left[0] + left[1]) + (left[2] + left[3]);
    }
    sum = vf_wave_sum(sum);
    if ((tid & 63) == 0) ss[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) vf_sums(a, b)[blockIdx.x] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
}

// From a refused draft on: its siblings, and the token.  (A sibling that is taken leads on to nodes whose rows may not have been
// looked at, and to other sums: this workgroup then does both by itself.)
__global__ void __launch_bounds__(VF_W) k_verify_rest(VerifyArgs a) {
    __shared__ VfShared S;
    const int b = blockIdx.x, tid = threadIdx.x, T = a.T;
    const VfState state = *vf_state(a, b);
    if (state.status != VF_LEFT) return;
    const VfScale s = vf_scale(a, b);
    vf_put(S, a, vf_draft(a, b));
    if (tid == 0) S.m[state.cur] = state.m, S.top_at[state.cur] = state.first, S.sum[state.cur] = 1.0 / state.per;
    __syncthreads();
    int* path = a.path + (int64_t)b * T;
    int cur = state.cur, n = state.n, past = state.child;
    VfLeft f = vf_at(S, a, b, cur);
    f.per = state.per;
    f.q = a.draft + ((int64_t)b * T + cur) * a.ldd;
    f.a = 1.0;
    const double* sums = vf_sums(a, b);
    double left = vf_sum(S, [&](int i) { return sums[i]; }, a.slices);
    bool summed = true;                                        // sums are those of what is left
    for (;;) {
        int next = -1;
        if (S.sum[cur] > 0.0)
            for (uint64_t children = vf_children(S, T, cur, past); children; children &= children - 1) {
                const int c = __builtin_ctzll(children);
                const double q = (double)S.q[c];
                if ((double)S.u[c] * left * q < fmax(vf_child(S, s, f, c) * f.per - f.a * q, 0.0)) {
                    next = c;
                    break;
                }
                f.a += left;
                f.q = a.draft + ((int64_t)b * T + cur) * a.ldd;
                left = vf_sum(S, [&](int i) { return vf_left(S, s, f, i); }, a.V);
                summed = false;
            }
        if (next < 0) break;
        cur = next, past = 0;
        n++;
        if (tid == 0) path[n] = next;
        vf_row_anew(S, a, s, b, cur);
        f = vf_at(S, a, b, cur);
        left = 1.0;
        summed = false;
    }
    int token = -1;
    if (S.sum[cur] > 0.0) {
        if (!(left > 0.0)) {                                   // nothing is left: drawn from p itself
            f.q = nullptr, f.a = 0.0;
            summed = false;
        }
        token = vf_draw(S, a, s, f, left, nullptr, sums, !summed);
    }
    for (int i = n + 1 + tid; i < T; i += VF_W) path[i] = -1;
    if (tid == 0) a.accepted[b] = n, a.token[b] = token;
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// The states, the slices' statistics of every row and a row of sums for each request, for the smallest slices.
size_t verify_workspace(int B, int T, int V) {
    const size_t slices = ((size_t)V + VF_LEAST - 1) / VF_LEAST;
    return up256(B * sizeof(VfState)) + up256((size_t)B * T * slices * sizeof(VerifyPart)) + up256(B * slices * sizeof(double));
}

void launch_verify(const VerifyArgs& args, hipStream_t s) {
    VerifyArgs a = args;
    // Rows of a round: 8 nodes of each request, fewer where those are more than 64 MB, and in the last round whatever is left.  All at
    // once where there are no more than 8 nodes (of up to 240 MB), or 24 of 64 MB in all: one round then costs less than the launches and
    // waits of several.  Measured, all at once and by this rule's rounds: 32 chains of 8 over 151936 ids (148 MB) 63 and 75 us, 48
    // with drawn drafts (223 MB) 112 and 116, but 64 chains (297 MB) 100 to 111 and 99; 8 trees of 10 (46 MB) 33 and 51, 4 of 24 (56 MB) 43 and 50; but 8 chains of 16 (74 MB) 44 and 41; one tree of 64
    // (37 MB) 65 and 29, four (148 MB) 86 and 44; 16 of 64 over 16000 ids (62 MB) 125 and 75, over 32000 (125 MB) 146 and 69.  Of 16 nodes a
    // request in place of 8 the last two take 79 and 77; of 4, four trees of 64 take 52 and 64 chains of 16 over 32000 ids 68, as with 8 (70).
    // More than 64 MB a round: 16 trees of 64 over 248320 ids 90 us, 101 with 128 MB.
    const int64_t row_bytes = (int64_t)a.B * a.V * 4, all_bytes = row_bytes * a.T, fit = std::min<int64_t>(8, (64 << 20) / row_bytes);
    const bool once = all_bytes <= (64 << 20) ? a.T <= 24 : a.T <= 8 && all_bytes <= (240 << 20);
    const int most = once || fit >= a.T ? a.T : fit < 1 ? 1 : (int)fit, rounds = most < a.T ? VF_ROUNDS : 1;
    // the largest slice that leaves two workgroups a CU in the first round
    a.slice = VF_MOST;
    while (a.slice > VF_LEAST && (int64_t)a.B * most * ((a.V + a.slice - 1) / a.slice) < 2 * device_cus()) a.slice /= 2;
    a.shift = __builtin_ctz((unsigned)a.slice);
    a.slices = (a.V + a.slice - 1) / a.slice;
    a.parts_at = up256(a.B * sizeof(VfState));
    a.sums_at = a.parts_at + up256((size_t)a.B * a.T * a.slices * sizeof(VerifyPart));
    auto al = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0; };
    const bool v4 = al(a.x, a.ldx) && (!a.draft || al(a.draft, a.ldd));
    const size_t lds = a.slice * sizeof(float), all = VF_MOST * sizeof(double);
    for (int round = 0; round < rounds; round++) {
        const int rows = round + 1 < rounds ? most : a.T;
        const dim3 grid(a.slices, a.B, rows < 4 ? rows : 4);
        auto stats = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(VF_T), lds, s, a, round, rows); };
        if (a.slice == 4096) v4 ? stats(k_verify_stats<true, 4096>) : stats(k_verify_stats<false, 4096>);
        else v4 ? stats(k_verify_stats<true, 2048>) : stats(k_verify_stats<false, 2048>);
        hipLaunchKernelGGL(k_verify_walk, dim3(a.B), dim3(VF_W), all, s, a, round, rows);
    }
    if (!a.draft) return;
    auto sums = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.slices, a.B), dim3(VF_T), 2 * lds, s, a); };
    if (a.slice == 4096) v4 ? sums(k_verify_left<true, 4096>) : sums(k_verify_left<false, 4096>);
    else v4 ? sums(k_verify_left<true, 2048>) : sums(k_verify_left<false, 2048>);
    hipLaunchKernelGGL(k_verify_rest, dim3(a.B), dim3(VF_W), all + VF_MOST * sizeof(float), s, a);
}

}  // namespace kq
