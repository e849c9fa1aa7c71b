// Penalties, biases and a grammar mask on the requests' logits, with the greedy pick (include/kq.h:
// kq_logits_penalize).
//
// A workgroup takes a slice of one row's vocabulary.  The history and the bias list name few ids anywhere in the row, so
// each workgroup scans them once and notes in LDS, per id of its slice, how often it occurs after the prompt, whether
// it occurs at all (integer atomics: any order gives the same) and its last bias entry.  Then one pass over the
// slice's logits applies the steps and keeps the best; the pick folds into one key per row, as argmax_block.h does
// for a single row.
#include "argmax_block.h"
#include "kq_internal.h"

namespace kq {

constexpr int LG_SLICE = 4096;               // ids of a workgroup: 32 KB of LDS for the two notes
constexpr uint32_t LG_SEEN = 0x80000000u;    // the id occurs; the low bits count occurrences after the prompt
constexpr int LG_ROW_BYTES = 2 * ARG_LINE;   // workspace of a row: the key's line, the ticket's line

template <bool V4>
__global__ void __launch_bounds__(256) k_logits(LogitsArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t note[LG_SLICE], bias[LG_SLICE];
    __shared__ ArgBest wave_best[4];
    const int b = blockIdx.y, v0 = blockIdx.x * LG_SLICE, nv = min(LG_SLICE, a.V - v0), tid = threadIdx.x;
    const int nh = a.hist ? min(max(a.hist_len[b], 0), a.max_hist) : 0, nb = a.bias_id ? a.nb : 0;
    if (nh | nb) {
        for (int i = 4 * tid; i < LG_SLICE; i += 1024) {
            *reinterpret_cast<u32x4*>(note + i) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(bias + i) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
        const int prompt = a.prompt_len ? a.prompt_len[b] : 0;
        const int32_t* hist = a.hist + (int64_t)b * a.ldh;
        for (int i = tid; i < nh; i += 256) {
            const uint32_t id = (uint32_t)hist[i] - (uint32_t)v0;
            if (id < (uint32_t)nv) {
                atomicOr(&note[id], LG_SEEN);
                if (i >= prompt) atomicAdd(&note[id], 1u);
            }
        }
        for (int i = tid; i < nb; i += 256) {
            const uint32_t id = (uint32_t)a.bias_id[(int64_t)b * a.ldb + i] - (uint32_t)v0;
            if (id < (uint32_t)nv) atomicMax(&bias[id], (uint32_t)i + 1u);
        }
        __syncthreads();
    }
    const float rep = a.rep ? a.rep[b] : 1.0f, freq = a.freq ? a.freq[b] : 0.0f, pres = a.pres ? a.pres[b] : 0.0f;
    const float* x = a.x + (int64_t)b * a.ldx + v0;
    float* y = a.y ? a.y + (int64_t)b * a.ldy + v0 : nullptr;
    const uint32_t* allowed = a.allowed ? a.allowed + (int64_t)b * a.ldm + (v0 >> 5) : nullptr;
    ArgBest best{-1e30f, -1};
    auto step = [&](float t, uint32_t seen, uint32_t entry, bool ok) {
        if (seen) {
            if (a.rep) t = t > 0.0f ? t / rep : t * rep;
            const uint32_t c = seen & ~LG_SEEN;
            if (c) {
                t = t - freq * (float)c;
                t = t - pres;
            }
        }
        if (entry) t = t + a.bias_val[(int64_t)b * a.ldb + entry - 1];
        return ok ? t : -INFINITY;
    };
    auto allowed_at = [&](int i) { return allowed ? allowed[i >> 5] >> (i & 31) : ~0u; };
    auto one = [&](int i) {
        const float t = step(x[i], nh ? note[i] : 0u, nb ? bias[i] : 0u, allowed_at(i) & 1u);
        if (y) y[i] = t;
        arg_take(best, t, v0 + i);
    };
    if constexpr (V4) {
        const u32x4 none = {0, 0, 0, 0};
        for (int i = 4 * tid; i + 3 < nv; i += 1024) {
            f32x4 t = *reinterpret_cast<const f32x4*>(x + i);
            const u32x4 n4 = nh ? *reinterpret_cast<const u32x4*>(note + i) : none;
            const u32x4 b4 = nb ? *reinterpret_cast<const u32x4*>(bias + i) : none;
            const uint32_t ok = allowed_at(i);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                t[k] = step(t[k], n4[k], b4[k], (ok >> k) & 1u);
                arg_take(best, t[k], v0 + i + k);
            }
            if (y) *reinterpret_cast<f32x4*>(y + i) = t;
        }
        for (int i = (nv & ~3) + tid; i < nv; i += 256) one(i);
    } else {
        for (int i = tid; i < nv; i += 256) one(i);
    }
    if (!a.picked) return;
    best = arg_wave_reduce(best);
    if ((tid & 63) == 0) wave_best[tid >> 6] = best;
    __syncthreads();
    if (tid) return;
    for (int w = 0; w < 4; w++) best = arg_combine(best, wave_best[w]);
    // fold into the row's key; whoever takes the row's last ticket reads the key and clears both
    auto* key = reinterpret_cast<unsigned long long*>(a.ws + (size_t)b * LG_ROW_BYTES);
    auto* ticket = reinterpret_cast<unsigned int*>(a.ws + (size_t)b * LG_ROW_BYTES + ARG_LINE);
    atomicMax(key, arg_key(best));
    __builtin_amdgcn_s_waitcnt(0x0f70);                  // vmcnt(0): the max has completed
    if (atomicAdd(ticket, 1u) != gridDim.x - 1) return;
    a.picked[b] = (int32_t)(0xffffffffu - (uint32_t)atomicExch(key, 0ull));
    atomicExch(ticket, 0u);
}

size_t logits_workspace(int B) { return (size_t)B * LG_ROW_BYTES; }

void launch_logits(const LogitsArgs& a, hipStream_t s) {
    const dim3 grid((a.V + LG_SLICE - 1) / LG_SLICE, a.B);
    auto al = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0; };
    if (al(a.x, a.ldx) && (!a.y || al(a.y, a.ldy))) hipLaunchKernelGGL(k_logits<true>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_logits<false>, grid, dim3(256), 0, s, a);
}

}  // namespace kq
