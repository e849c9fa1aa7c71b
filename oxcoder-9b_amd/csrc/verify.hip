// Verification of drafted tokens against the target's probabilities, from given random numbers (include/kq.h: kq_verify).
//
// With p the softmax of a node's row and q the probabilities that its children were drawn from, refusing a child leaves
// max(p - q, 0) normalised, refusing another max of that less q, and so on: after k refusals max(p - a q, 0) / Z with
// a_0 = 0, Z_0 = 1, a_k+1 = a_k + Z_k, Z_k+1 = sum max(p - a_k+1 q, 0).  So what is left is one number a and the row.  For a
// child that was not drawn (q holds it alone) what is left is p without the refused tokens.
//
// The first kernel takes every row's softmax statistics slice by slice; the second, one workgroup a request, walks the tree on
// the rows' statistics and its tokens' logits, all fetched at once, and draws the next token: over the slices' sums, then
// inside one slice.
#include "kq_device.h"
#include "kq_internal.h"

namespace kq {

constexpr int VF_T = 256;                    // threads of the first kernel
constexpr int VF_MOST = 8192;                // ids of its largest slice
constexpr int VF_LEAST = 2048;
constexpr int VF_W = 1024;                   // threads of the second

// Weights are held in 64 bits as well: a vocabulary's running sum has a border for every id, and fp32 weights, off by 2^-24
// each, would put one draw in some hundred on the border's other side.
struct VfScale {
    double c;                  // log2(e) / temperature
    bool greedy;               // temperature 0: the first of the largest logits alone
};
__device__ __forceinline__ VfScale vf_scale(const VerifyArgs& a, int b) {
    const float t = a.temperature ? a.temperature[b] : 1.0f;
    const bool greedy = !(t > 0.0f);
    return VfScale{greedy ? 0.0 : 1.4426950408889634 / (double)t, greedy};
}
// 2^z, z <= 0: ln(2)^k / k! f^k summed to k = 11 over the fraction f in -1/2..1/2, off by at most (ln(2)/2)^12 / 12! = 6.3e-15
// of it; below 2^-1000, and for a NaN, 0.
__device__ __forceinline__ double vf_exp2(double z) {
    if (!(z > -1000.0)) return 0.0;
    const double n = rint(z), f = z - n;
    double p = 4.44553827187081e-10;
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    return ldexp(fma(p, f, 1.0), (int)n);
}
// x's weight beside the largest logit m: 1 for m itself, 0 for -inf and NaN.
__device__ __forceinline__ double vf_weight(const VfScale& s, float x, float m) {
    return x == m ? 1.0 : vf_exp2(((double)x - (double)m) * s.c);
}

__device__ __forceinline__ double vf_wave_sum(double v) {
    for (int w = 32; w; w >>= 1) v += __shfl_xor(v, w, 64);
    return v;
}

template <bool V4>
__global__ void __launch_bounds__(VF_T) k_verify_stats(VerifyArgs a) {
    __shared__ float sm[VF_T / 64];
    __shared__ double ss[VF_T / 64];
    __shared__ int sa[VF_T / 64];
    const int64_t row = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, v0 = blockIdx.x * a.slice, nv = min(a.slice, a.V - v0);
    const float* x = a.x + row * a.ldx + v0;
    const VfScale s = vf_scale(a, (int)(row / a.T));
    f32x4 v[VF_MOST / VF_T / 4];
#pragma unroll
    for (int n = 0; n < VF_MOST / VF_T / 4; n++) {
        const int i = 4 * (n * VF_T + tid);
        v[n] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 3 < nv) {
            if constexpr (V4) v[n] = *reinterpret_cast<const f32x4*>(x + i);
            else v[n] = *reinterpret_cast<const f32x4_a4*>(x + i);
        } else {
            for (int k = 0; k < 3; k++)
                if (i + k < nv) v[n][k] = x[i + k];
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int n = 0; n < VF_MOST / VF_T / 4; n++) m = fmaxf(m, fmaxf(fmaxf(v[n].x, v[n].y), fmaxf(v[n].z, v[n].w)));
    for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
    if (lane == 0) sm[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    double sum = 0.0;
    int at = INT_MAX;
#pragma unroll
    for (int n = VF_MOST / VF_T / 4 - 1; n >= 0; n--)
#pragma unroll
        for (int k = 3; k >= 0; k--) {
            if (v[n][k] == m) at = 4 * (n * VF_T + tid) + k;
            if (m > -INFINITY) sum += vf_weight(s, v[n][k], m);
        }
    sum = vf_wave_sum(sum);
    for (int w = 32; w; w >>= 1) at = min(at, __shfl_xor(at, w, 64));
    if (lane == 0) ss[wave] = sum, sa[wave] = at;
    __syncthreads();
    if (tid) return;
    VerifyPart* part = reinterpret_cast<VerifyPart*>(a.ws) + row * a.slices + blockIdx.x;
    at = min(min(sa[0], sa[1]), min(sa[2], sa[3]));
    *part = VerifyPart{(ss[0] + ss[1]) + (ss[2] + ss[3]), m, m > -INFINITY ? v0 + at : 0};
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
    double sum[TREE_MOST];
    double seg[VF_W], wave[VF_W / 64];
    int found;
};

__device__ __forceinline__ double vf_left(const VfShared& S, const VfScale& s, const VfLeft& f, int i) {
    const double e = s.greedy ? (i == f.first ? 1.0 : 0.0) : vf_weight(s, f.x[i], f.m);
    if (f.q) return fmax(e * f.per - f.a * (double)f.q[i], 0.0);
    for (int k = 0; k < f.gone; k++)
        if (S.refused[k] == i) return 0.0;
    return e;
}

// Sums of the row's segments of `len` ids into S.seg, and their total.
__device__ double vf_segments(VfShared& S, const VfScale& s, const VfLeft& f, int V, int len) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (V + len - 1) / len;
    __syncthreads();
    for (int g = wave; g < n; g += VF_W / 64) {
        const int end = min((g + 1) * len, V);
        double sum = 0.0;
        for (int i = g * len + lane; i < end; i += 64) sum += vf_left(S, s, f, i);
        sum = vf_wave_sum(sum);
        if (lane == 0) S.seg[g] = sum;
    }
    __syncthreads();
    double total = 0.0;
    for (int g = lane; g < n; g += 64) total += S.seg[g];
    return vf_wave_sum(total);
}

// The smallest id of [from, to) at which before + the running sum exceeds the target; the last one with a weight where
// none does (the sums' own rounding), -1 where none has one.
__device__ int vf_pick(VfShared& S, const VfScale& s, const VfLeft& f, int from, int to, double before, double target) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int last = -1;
    for (int i0 = from; i0 < to; i0 += VF_W) {
        const int i = i0 + tid;
        const double w = i < to ? vf_left(S, s, f, i) : 0.0;
        double run = w;
        for (int k = 1; k < 64; k <<= 1) {
            const double y = __shfl_up(run, k, 64);
            if (lane >= k) run += y;
        }
        __syncthreads();
        if (tid == 0) S.found = INT_MAX;
        if (lane == 63) S.wave[wave] = run;
        __syncthreads();
        double ahead = before;
        for (int k = 0; k < wave; k++) ahead += S.wave[k];
        if (w > 0.0 && ahead + run > target) atomicMin(&S.found, i);
        const uint64_t some = __ballot(w > 0.0);
        if (some) last = i0 + 64 * wave + 63 - __builtin_clzll(some);
        for (int k = 0; k < VF_W / 64; k++) before += S.wave[k];
        __syncthreads();
        if (S.found != INT_MAX) return S.found;
    }
    __syncthreads();
    if (tid == 0) S.found = -1;
    __syncthreads();
    if (lane == 0) atomicMax(&S.found, last);
    __syncthreads();
    return S.found;
}

__global__ void __launch_bounds__(VF_W) k_verify_walk(VerifyArgs a) {
    __shared__ VfShared S;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, T = a.T;
    const VfScale s = vf_scale(a, b);
    const int64_t row0 = (int64_t)b * T;
    const VerifyPart* parts = reinterpret_cast<const VerifyPart*>(a.ws) + row0 * a.slices;
    if (tid < T) {
        const int up = a.parents[(int64_t)b * a.ldp + tid], tok = a.tokens[(int64_t)b * a.ldt + tid];
        const bool ok = up >= 0 && up < tid, in = ok && tok >= 0 && tok < a.V;
        S.tok[tid] = in ? tok : -1;
        S.up[tid] = tid == 0 ? up : ok ? up : -2;
        S.u[tid] = a.uniform[(int64_t)b * a.ldu + tid];
        S.x[tid] = in ? a.x[(row0 + up) * a.ldx + tok] : -INFINITY;
        S.q[tid] = in && a.draft ? a.draft[(row0 + up) * a.ldd + tok] : 0.0f;
    }
    // every row's statistics: the slices' brought to the row's largest logit
    for (int t = wave; t < T; t += VF_W / 64) {
        const VerifyPart* p = parts + (int64_t)t * a.slices;
        float m = -INFINITY;
        for (int i = lane; i < a.slices; i += 64) m = fmaxf(m, p[i].m);
        for (int w = 32; w; w >>= 1) m = fmaxf(m, __shfl_xor(m, w, 64));
        double sum = 0.0;
        int at = INT_MAX;
        for (int i = lane; i < a.slices; i += 64) {
            const VerifyPart y = p[i];
            if (y.m == m) at = min(at, y.at);
            sum += y.sum * vf_weight(s, y.m, m);
        }
        sum = vf_wave_sum(sum);
        for (int w = 32; w; w >>= 1) at = min(at, __shfl_xor(at, w, 64));
        if (lane == 0) S.m[t] = m, S.sum[t] = m == -INFINITY ? 0.0 : s.greedy ? 1.0 : sum, S.top_at[t] = at;
    }
    __syncthreads();
    int* path = a.path + row0;
    const int seg_len = ((a.V + VF_W - 1) / VF_W + 255) / 256 * 256;
    int cur = 0, n = 0;
    VfLeft f = {};
    double left = 0.0;
    if (S.up[0] == -1) {
        if (tid == 0) path[0] = 0;
        for (;;) {
            f = VfLeft{a.x + (row0 + cur) * a.ldx, nullptr, S.m[cur], S.top_at[cur], 0.0, 0.0, 0};
            left = S.sum[cur];
            int next = -1;
            if (left > 0.0) {
                f.per = 1.0 / left;
                if (a.draft) left = 1.0;
                uint64_t children = __ballot(lane < T && lane > 0 && S.up[lane < T ? lane : 0] == cur);
                for (; children; children &= children - 1) {
                    const int c = __builtin_ctzll(children), tok = S.tok[c];
                    if (tok < 0) continue;                     // no token: refused, and nothing leaves
                    const double e = s.greedy ? (tok == f.first ? 1.0 : 0.0) : vf_weight(s, S.x[c], f.m);
                    if (a.draft) {
                        const double q = (double)S.q[c];
                        if ((double)S.u[c] * left * q < fmax(e * f.per - f.a * q, 0.0)) next = c;
                        if (next >= 0) break;
                        f.a += left;
                        f.q = a.draft + (row0 + cur) * a.ldd;
                        left = vf_segments(S, s, f, a.V, seg_len);
                    } else {
                        bool again = false;                    // refused already: it holds nothing any more
                        for (int k = 0; k < f.gone; k++) again |= S.refused[k] == tok;
                        const double w = again ? 0.0 : e;
                        if ((double)S.u[c] * left < w) next = c;
                        if (next >= 0) break;
                        left -= w;
                        __syncthreads();
                        if (tid == 0) S.refused[f.gone] = tok;
                        __syncthreads();
                        f.gone++;
                    }
                }
            }
            if (next < 0) break;
            cur = next;
            n++;
            if (tid == 0) path[n] = next;
            __syncthreads();
        }
    } else {
        n = -1;
    }
    for (int i = n + 1 + tid; i < T; i += VF_W) path[i] = -1;
    int token = -1;
    if (n >= 0 && S.sum[cur] > 0.0) {
        if (!(left > 0.0)) f.q = nullptr, f.a = 0.0, f.gone = 0;   // nothing is left: drawn from p itself
        left = vf_segments(S, s, f, a.V, seg_len);
        const double target = (double)S.u[0] * left;
        // the first segment at which the running sum exceeds the target
        const int segs = (a.V + seg_len - 1) / seg_len;
        double run = 0.0, ahead = 0.0;
        int at = -1, last = -1;
        for (int g = 0; g < segs; g++) {
            const double w = S.seg[g];
            if (w > 0.0) {
                last = g;
                if (at < 0 && run + w > target) at = g, ahead = run;
            }
            run += w;
        }
        if (at < 0) {
            at = last;
            ahead = -1.0;                                      // (rounding: whatever comes last)
        }
        if (at >= 0) token = vf_pick(S, s, f, at * seg_len, min((at + 1) * seg_len, a.V), ahead < 0.0 ? 0.0 : ahead, ahead < 0.0 ? INFINITY : target);
    }
    if (tid == 0) {
        a.accepted[b] = n;
        a.token[b] = token;
    }
}

static int vf_slice(int B, int T, int V) {
    (void)B, (void)T;
    return V <= VF_LEAST ? VF_LEAST : VF_MOST;
}

size_t verify_workspace(int B, int T, int V) {
    const int slice = vf_slice(B, T, V);
    return ((size_t)B * T * ((V + slice - 1) / slice) * sizeof(VerifyPart) + 255) & ~(size_t)255;
}

void launch_verify(const VerifyArgs& args, hipStream_t s) {
    VerifyArgs a = args;
    a.slice = vf_slice(a.B, a.T, a.V);
    a.slices = (a.V + a.slice - 1) / a.slice;
    auto go = [&](auto kernel, dim3 grid, int threads) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, a); };
    const bool v4 = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx % 4 == 0;
    go(v4 ? k_verify_stats<true> : k_verify_stats<false>, dim3(a.slices, a.B * a.T), VF_T);
    go(k_verify_walk, dim3(a.B), VF_W);
}

}  // namespace kq
