// Trees of drafted tokens in a paged cache: what a tree's parents say of its nodes, once a step for all layers, and the
// accepted nodes' entries moved together (include/kq.h: kq_tree_plan, kq_kv_keep).
#include "kv_device.h"

namespace kq {

// One wave per request, a lane per node.  A node's word of ancestors doubles its reach in each of six steps: it takes up
// the word of the node that its link points to, and that node's link.  A launch's latency, 2 to 3 us, once for all layers.
__global__ void __launch_bounds__(64) k_tree_plan(TreeArgs a) {
    const int b = blockIdx.x, t = threadIdx.x;
    const int up = t < a.T ? a.parents[(int64_t)b * a.ldp + t] : -2, base = a.base[b];
    int bad = up < -1 || up >= t, link = bad ? -1 : up;
    uint32_t lo = t < 32 ? 1u << t : 0u, hi = t < 32 ? 0u : 1u << (t - 32);
    for (int i = 0; i < 6; i++) {
        const int from = max(link, 0);
        const uint32_t l = __shfl(lo, from, 64), h = __shfl(hi, from, 64);
        const int x = __shfl(bad, from, 64), on = __shfl(link, from, 64);
        if (link >= 0) lo |= l, hi |= h, bad |= x, link = on;
    }
    if (t >= a.T) return;
    const int64_t n = (int64_t)b * a.T + t;
    const bool there = !bad && base >= 0 && base <= (1 << 30);
    a.seen[n] = bad ? 0 : (uint64_t)hi << 32 | lo;
    a.seq[n] = there ? b : -1;
    a.pos[n] = there ? base + __popc(lo) + __popc(hi) - 1 : -1;
    a.slot[n] = there ? base + t : -1;
}

void launch_tree_plan(const TreeArgs& a, int seqs, hipStream_t s) {
    hipLaunchKernelGGL(k_tree_plan, dim3(seqs), dim3(64), 0, s, a);
}

// A thread holds one 16-byte piece of an entry, of k or of v (past those, one scale), and moves it for each node of the
// path in turn.  A path rises, so an entry's new place lies below every place that a later node comes from: moved in order,
// nothing is overwritten before it was read.  Bound by the chain of path, table and data for one request (3.8 us for 32 layers of 3
// nodes, one launch for all of them), by memory for many (64 requests of 6 nodes: 59 MB in 10.8 us, 5.4 TB/s).
__global__ void __launch_bounds__(256) k_kv_keep(KeepArgs a) {
    const KeepLayer& L = a.layer[blockIdx.z];
    const int b = blockIdx.y, lane = threadIdx.x & 63;
    const int per = L.row / 16, half = L.heads * per, scales = L.k_scale ? 2 * L.heads : 0;
    // lane i: the path's node i, where it lies and where it goes
    const int at = lane < a.T ? a.path[(int64_t)b * a.ldp + lane] : -1, before = __shfl_up(at, 1, 64);
    const int base = a.base[b];
    const uint64_t good = __ballot(at >= lane && at < a.T && (lane == 0 || at > before));
    const int n = ~good ? __builtin_ctzll(~good) : 64;
    const int64_t from = (int64_t)base + at, to = (int64_t)base + lane;
    bool moves = lane < n && at > lane && base >= 0 && from < a.table.cap;
    int from_page = -1, to_page = -1;
    if (moves) {
        const int32_t* table = a.table.pages + (int64_t)b * a.table.ld;
        from_page = table[from / a.page_size];
        to_page = table[to / a.page_size];
    }
    moves = moves && (unsigned)from_page < (unsigned)a.pages && (unsigned)to_page < (unsigned)a.pages;
    const int from_off = (int)(from & (a.page_size - 1)), to_off = (int)(to & (a.page_size - 1));
    const uint64_t some = __ballot(moves);
    const int pieces = 2 * half + scales;
    // The loops are the same for a wave's lanes, as each takes its entries' places from all of them: what a lane without a
    // piece of its own holds must be there too.
    for (int i0 = blockIdx.x * 256 + __builtin_amdgcn_readfirstlane(threadIdx.x & ~63); i0 < pieces; i0 += gridDim.x * 256) {
        const int i = min(i0 + lane, pieces - 1);
        const bool live = i0 + lane < pieces, scale = i >= 2 * half;
        const int j = scale ? i - 2 * half : i, is_v = j >= (scale ? L.heads : half), h = is_v ? j - (scale ? L.heads : half) : j;
        uint8_t* p;
        int64_t page, pos;
        if (scale) {
            p = reinterpret_cast<uint8_t*>((is_v ? L.v_scale : L.k_scale) + h * L.scale_head);
            page = 4 * L.scale_page, pos = 4 * L.scale_pos;
        } else {
            p = (is_v ? L.v : L.k) + h / per * L.head + h % per * 16;
            page = L.page, pos = L.pos;
        }
        for (uint64_t todo = some; todo; todo &= todo - 1) {
            const int k = __builtin_ctzll(todo);
            const int sp = __builtin_amdgcn_readlane(from_page, k), so = __builtin_amdgcn_readlane(from_off, k);
            const int dp = __builtin_amdgcn_readlane(to_page, k), d = __builtin_amdgcn_readlane(to_off, k);
            if (!live) continue;
            const uint8_t* src = p + sp * page + so * pos;
            uint8_t* dst = p + dp * page + d * pos;
            if (scale) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
            else *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
        }
    }
}

void launch_kv_keep(const KeepArgs& a, int layers, int seqs, hipStream_t s) {
    int most = 1;
    for (int i = 0; i < layers; i++) {
        const KeepLayer& L = a.layer[i];
        most = max(most, 2 * L.heads * (L.row / 16) + (L.k_scale ? 2 * L.heads : 0));
    }
    hipLaunchKernelGGL(k_kv_keep, dim3((most + 255) / 256, seqs, layers), dim3(256), 0, s, a);
}

}  // namespace kq
