// Penalties, biases and a grammar mask on the requests' logits, with the greedy pick (include/kq.h:
// kq_logits_penalize).
//
// A workgroup takes a slice of one row's vocabulary, its logits and mask on their way to registers from the start.  The
// history and the bias list name few ids anywhere in the row, so each workgroup scans them once and notes in LDS, per id of its
// slice, how often it occurs after the prompt, whether it occurs at all and its last bias entry (integer atomics: any
// order gives the same).  Then every thread steps its logits and keeps the best.  The pick folds into one key per row, as
// argmax_block.h does for a single row.
//
// 128 rows of 248320 with histories of 4000, 20 biases and a mask: 260 MB in 55 us, 4.7 TB/s, a large copy's rate.  Listing the noted ids
// and stepping them packed, ahead of the pass, took 79 us: it read their logits a second time, one round trip later.
// 32 rows of 151936: 12 us (39 MB), 608 workgroups on 256 CUs and one scan's latency; halving the slices scans more (15 us).
// One row: 5.5 us, the launch and the chain of list, barrier, logits and the pick's two atomics.
#include "argmax_block.h"
#include "kq_internal.h"

namespace kq {

constexpr int LG_T = 512;                    // threads
constexpr int LG_STEP = 4 * LG_T;            // ids of a workgroup's pass of 16-byte loads
constexpr int LG_AHEAD = 4;                  // history ids a thread fetches ahead
constexpr int LG_MOST = 4 * LG_STEP;         // ids of the largest slice: 32 KB of notes, four workgroups a CU
// A note: the last bias entry + 1, whether the id occurs, occurrences after the prompt.
constexpr int LG_ENTRY = 21, LG_COUNT = 20;
constexpr uint32_t LG_SEEN = 1u << LG_COUNT;
constexpr int LG_MOST_HIST = 1 << LG_COUNT, LG_MOST_BIAS = 1 << (32 - LG_ENTRY);
constexpr int LG_ROW_BYTES = 2 * ARG_LINE;   // workspace of a row: the key's line, the ticket's line

// A row's penalties.
struct LgRow {
    float rep, freq, pres;
    bool has_rep, has_freq, has_pres;
};
__device__ __forceinline__ LgRow lg_row(const LogitsArgs& a, int b) {
    return LgRow{a.rep ? a.rep[b] : 1.0f, a.freq ? a.freq[b] : 0.0f, a.pres ? a.pres[b] : 0.0f, a.rep != nullptr, a.freq != nullptr,
                 a.pres != nullptr};
}
// t after the penalties, each step rounded.
__device__ __forceinline__ float lg_step(const LgRow& r, float t, bool seen, uint32_t count) {
    if (seen && r.has_rep) t = t > 0.0f ? t / r.rep : t * r.rep;
    if (count && r.has_freq) t = t - r.freq * (float)count;
    if (count && r.has_pres) t = t - r.pres;
    return t;
}

// Folds the workgroup's best into the row's key; whoever takes the row's last ticket reads the key and clears both.
__device__ __forceinline__ void lg_finish(const LogitsArgs& a, int b, ArgBest best) {
    __shared__ ArgBest wave_best[LG_T / 64];
    best = arg_wave_reduce(best);
    if ((threadIdx.x & 63) == 0) wave_best[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 0; w < LG_T / 64; w++) best = arg_combine(best, wave_best[w]);
    auto* key = reinterpret_cast<unsigned long long*>(a.ws + (size_t)b * LG_ROW_BYTES);
    auto* ticket = reinterpret_cast<unsigned int*>(a.ws + (size_t)b * LG_ROW_BYTES + ARG_LINE);
    atomicMax(key, arg_key(best));
    __builtin_amdgcn_s_waitcnt(0x0f70);                  // vmcnt(0): the max has completed
    if (atomicAdd(ticket, 1u) != gridDim.x - 1) return;
    a.picked[b] = (int32_t)(0xffffffffu - (uint32_t)atomicExch(key, 0ull));
    atomicExch(ticket, 0u);
}

template <bool V4>
__global__ void __launch_bounds__(LG_T) k_logits(LogitsArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t note[];       // [slice], then the biases [nb]
    float* const bias = reinterpret_cast<float*>(note + a.slice);
    const int b = blockIdx.y, v0 = blockIdx.x * a.slice, nv = min(a.slice, a.V - v0), tid = threadIdx.x;
    const float* x = a.x + (int64_t)b * a.ldx + v0;
    const uint32_t* allowed = a.allowed ? a.allowed + (int64_t)b * a.ldm + (v0 >> 5) : nullptr;
    f32x4 t[LG_MOST / LG_STEP];
    uint32_t ok[LG_MOST / LG_STEP];
#pragma unroll
    for (int n = 0; n < LG_MOST / LG_STEP; n++) {
        const int i = n * LG_STEP + 4 * tid;
        ok[n] = ~0u;
        if (i + 3 < nv) {
            if constexpr (V4) t[n] = *reinterpret_cast<const f32x4*>(x + i);
            else t[n] = *reinterpret_cast<const f32x4_a4*>(x + i);
            if (allowed) ok[n] = allowed[i >> 5];
        }
    }
    // the lists' first entries as well, read before the history's length is known: its row holds max_hist ids
    const int32_t* hist = a.hist + (int64_t)b * a.ldh;
    const int64_t bias0 = (int64_t)b * a.ldb;
    const int held = a.hist ? a.max_hist : 0, nb = a.bias_id ? a.nb : 0;
    uint32_t id[LG_AHEAD], bias_id = ~0u;
    float bias_val = 0.0f;
#pragma unroll
    for (int k = 0; k < LG_AHEAD; k++) id[k] = tid + k * LG_T < held ? (uint32_t)hist[tid + k * LG_T] : ~0u;
    if (tid < nb) {
        bias_id = (uint32_t)a.bias_id[bias0 + tid];
        bias_val = a.bias_val[bias0 + tid];
    }
    const LgRow row = lg_row(a, b);
    const int nh = a.hist ? min(max(a.hist_len[b], 0), a.max_hist) : 0;
    const bool notes = nh | nb;
    if (notes) {
        for (int i = 4 * tid; i < a.slice; i += LG_STEP) *reinterpret_cast<u32x4*>(note + i) = u32x4{0, 0, 0, 0};
        const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
        __syncthreads();
        auto occurs = [&](uint32_t v, int i) {
            const uint32_t at = v - (uint32_t)v0;
            if (at < (uint32_t)nv && i < nh) {
                atomicOr(&note[at], LG_SEEN);
                if (i >= prompt) atomicAdd(&note[at], 1u);
            }
        };
        auto biased = [&](uint32_t v, float value, int i) {
            bias[i] = value;
            const uint32_t at = v - (uint32_t)v0, entry = (uint32_t)(i + 1) << LG_ENTRY;
            if (at >= (uint32_t)nv) return;
            uint32_t old = note[at];
            while (old < entry) {                                          // the fields below may change meanwhile
                const uint32_t was = atomicCAS(&note[at], old, (old & ((1u << LG_ENTRY) - 1)) | entry);
                if (was == old) break;
                old = was;
            }
        };
        if (tid < nb) biased(bias_id, bias_val, tid);
        for (int i = tid + LG_T; i < nb; i += LG_T) biased((uint32_t)a.bias_id[bias0 + i], a.bias_val[bias0 + i], i);
#pragma unroll
        for (int k = 0; k < LG_AHEAD; k++) occurs(id[k], tid + k * LG_T);
        for (int i0 = tid + LG_AHEAD * LG_T; i0 < nh; i0 += 4 * LG_T) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = i0 + k * LG_T < nh ? (uint32_t)hist[i0 + k * LG_T] : ~0u;
#pragma unroll
            for (int k = 0; k < 4; k++) occurs(v[k], i0 + k * LG_T);
        }
        __syncthreads();
    }
    float* y = a.y ? a.y + (int64_t)b * a.ldy + v0 : nullptr;
    ArgBest best{-1e30f, -1};
    auto noted = [&](float u, uint32_t n) {
        if (n) {
            u = lg_step(row, u, n & LG_SEEN, n & (LG_SEEN - 1));
            const uint32_t entry = n >> LG_ENTRY;
            if (entry) u = u + bias[entry - 1];
        }
        return u;
    };
#pragma unroll
    for (int n = 0; n < LG_MOST / LG_STEP; n++) {
        const int i = n * LG_STEP + 4 * tid;
        if (i + 3 >= nv) continue;
        const u32x4 m = notes ? *reinterpret_cast<const u32x4*>(note + i) : u32x4{0, 0, 0, 0};
        const uint32_t bits = ok[n] >> (i & 31);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float u = t[n][k];
            u = noted(u, m[k]);
            u = (bits >> k) & 1u ? u : -INFINITY;
            t[n][k] = u;
            arg_take_ascending(best, u, v0 + i + k);
        }
        if (y) {
            if constexpr (V4) *reinterpret_cast<f32x4*>(y + i) = t[n];
            else *reinterpret_cast<f32x4_a4*>(y + i) = t[n];
        }
    }
    if (tid < (nv & 3)) {                                                  // the last one to three ids
        const int i = (nv & ~3) + tid;
        float u = noted(x[i], notes ? note[i] : 0u);
        if (allowed && !(allowed[i >> 5] >> (i & 31) & 1u)) u = -INFINITY;
        arg_take(best, u, v0 + i);
        if (y) y[i] = u;
    }
    if (a.picked) lg_finish(a, b, best);
}

// Histories or bias lists too long for a note's fields: two notes per id, and every id stepped in place.
constexpr int LG_WIDE = 4096;
__global__ void __launch_bounds__(LG_T) k_logits_wide(LogitsArgs a) {
    __shared__ uint32_t note[LG_WIDE], bias[LG_WIDE];
    const int b = blockIdx.y, v0 = blockIdx.x * LG_WIDE, nv = min(LG_WIDE, a.V - v0), tid = threadIdx.x;
    const int nh = a.hist ? min(max(a.hist_len[b], 0), a.max_hist) : 0, nb = a.bias_id ? a.nb : 0;
    for (int i = tid; i < LG_WIDE; i += LG_T) note[i] = bias[i] = 0;
    __syncthreads();
    const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
    for (int i = tid; i < nh; i += LG_T) {
        const uint32_t id = (uint32_t)a.hist[(int64_t)b * a.ldh + i] - (uint32_t)v0;
        if (id < (uint32_t)nv) {
            atomicOr(&note[id], 1u << 31);
            if (i >= prompt) atomicAdd(&note[id], 1u);
        }
    }
    for (int i = tid; i < nb; i += LG_T) {
        const uint32_t id = (uint32_t)a.bias_id[(int64_t)b * a.ldb + i] - (uint32_t)v0;
        if (id < (uint32_t)nv) atomicMax(&bias[id], (uint32_t)i + 1u);
    }
    __syncthreads();
    const LgRow row = lg_row(a, b);
    ArgBest best{-1e30f, -1};
    for (int i = tid; i < nv; i += LG_T) {
        float t = lg_step(row, a.x[(int64_t)b * a.ldx + v0 + i], note[i] != 0, note[i] & ~(1u << 31));
        if (bias[i]) t = t + a.bias_val[(int64_t)b * a.ldb + bias[i] - 1];
        if (a.allowed && !(a.allowed[(int64_t)b * a.ldm + ((v0 + i) >> 5)] >> ((v0 + i) & 31) & 1u)) t = -INFINITY;
        if (a.y) a.y[(int64_t)b * a.ldy + v0 + i] = t;
        arg_take(best, t, v0 + i);
    }
    if (a.picked) lg_finish(a, b, best);
}

size_t logits_workspace(int B) { return (size_t)B * LG_ROW_BYTES; }

void launch_logits(const LogitsArgs& args, hipStream_t s) {
    LogitsArgs a = args;
    if ((a.hist && a.max_hist >= LG_MOST_HIST) || (a.bias_id && a.nb >= LG_MOST_BIAS)) {
        hipLaunchKernelGGL(k_logits_wide, dim3((a.V + LG_WIDE - 1) / LG_WIDE, a.B), dim3(LG_T), 0, s, a);
        return;
    }
    // the largest slice that leaves two workgroups a CU: every slice scans the whole history
    a.slice = LG_MOST;
    while (a.slice > LG_STEP && (int64_t)a.B * ((a.V + a.slice - 1) / a.slice) < 2 * device_cus()) a.slice /= 2;
    const dim3 grid((a.V + a.slice - 1) / a.slice, a.B);
    const size_t lds = a.hist || a.bias_id ? ((size_t)a.slice + (a.bias_id ? a.nb : 0)) * 4 : 0;
    auto al = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0; };
    if (al(a.x, a.ldx) && (!a.y || al(a.y, a.ldy))) hipLaunchKernelGGL(k_logits<true>, grid, dim3(LG_T), lds, s, a);
    else hipLaunchKernelGGL(k_logits<false>, grid, dim3(LG_T), lds, s, a);
}

}  // namespace kq
