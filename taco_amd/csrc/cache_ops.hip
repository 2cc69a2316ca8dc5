// The KV cache's own operators, all in place: the rows of an accepted path moved behind the context, and the
// cut of a cache to its budget by accumulated attention weight. No counterpart in the reference.
#include "intmath.h"
#include "launch.h"

namespace hs {

// Row copies go in words of W bytes: 16 where the head dim and the caches allow it, else 4.
template <int W>
struct Word;
template <>
struct Word<16> {
    typedef v4i type;
};
template <>
struct Word<4> {
    typedef int32_t type;
};

// ---- commit ----------------------------------------------------------------------------------------
// Row ctx + i takes row ctx + path[i], i < accepted. path[i] >= i, so with the rows in ascending order a
// row is read before anything is written over it. One wave per (layer, K or V, stream, head) panel.
template <int W>
__global__ __launch_bounds__(256) void k_commit(CachePtrs c, CommitArgs a, int n_panels) {
    typedef typename Word<W>::type T;
    const int lane = threadIdx.x & 63, task = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (task >= 2 * n_panels) return;
    const int panel = task >> 1, per = a.b * a.h, layer = panel / per, sh = panel - layer * per, s = sh / a.h;
    const uint32_t cap = (uint32_t)a.cap;
    const uint32_t ctx = a.ctx[s] < cap ? a.ctx[s] : cap;
    uint32_t acc = a.accepted[s] < (uint32_t)a.t ? a.accepted[s] : (uint32_t)a.t;
    acc = acc < cap - ctx ? acc : cap - ctx;
    if (a.ctx_out && layer == 0 && a.first && (task & 1) == 0 && sh == s * a.h && lane == 0) a.ctx_out[s] = ctx + acc;
    int8_t *base = ((task & 1) ? c.v[layer] : c.k[layer]) + (size_t)sh * cap * a.hd;
    const int words = a.hd / W, rows = 64 / words, r = lane / words, w = lane - r * words;
    if (r >= rows) return;
    for (uint32_t i = r; i < acc; i += rows) {
        const uint32_t p = a.path[(size_t)s * a.t + i];
        if (p == i || p >= cap - ctx) continue;  // in place already; a row past the cache is left alone
        ((T *)(base + (size_t)(ctx + i) * a.hd))[w] = ((const T *)(base + (size_t)(ctx + p) * a.hd))[w];
    }
}

static bool wide_words(const CachePtrs &c, int layers, int hd) {
    uintptr_t bits = (uintptr_t)hd;
    for (int l = 0; l < layers; l++) bits |= (uintptr_t)c.k[l] | (uintptr_t)c.v[l];
    return bits % 16 == 0;
}

hipError_t launch_commit(const CachePtrs &c, int layers, const CommitArgs &a, hipStream_t stream) {
    const int panels = layers * a.b * a.h;
    if (panels <= 0) return hipSuccess;
    const dim3 grid((2 * panels + 3) / 4);
    if (wide_words(c, layers, a.hd)) launch_k(k_commit<16>, grid, dim3(256), 0, stream, c, a, panels);
    else launch_k(k_commit<4>, grid, dim3(256), 0, stream, c, a, panels);
    return hipGetLastError();
}

// ---- evict -----------------------------------------------------------------------------------------
// One workgroup per (layer, stream, head) panel of n > budget keys. The `heavy` = budget - recent largest
// masses of the first n - recent keys stay (ties: the lowest index), by a radix selection of the
// heavy-th largest value, eight bits at a time. Attention over integers does not depend on the order of the
// keys, so only what must move moves: a kept key below `heavy` stays where it is, and the a-th free place below it
// takes the a-th kept key from above; the recent rows follow in order. Sources of the first kind lie at or above
// `heavy` and places below, so these copies need no order; the recent rows move down tile by tile after them.

constexpr int EV_NT = 256;

// Exclusive prefix sum of v over the workgroup; total: the sum. `slots` holds a value per wave.
__device__ __forceinline__ int block_scan(int v, int *slots, int tid, int &total) {
    const int lane = tid & 63, w = tid >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) slots[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < EV_NT / 64; i++) {
        before += i < w ? slots[i] : 0;
        total += slots[i];
    }
    return before + x - v;
}

template <int W>
__global__ __launch_bounds__(EV_NT) void k_evict(CachePtrs c, EvictArgs a) {
    typedef typename Word<W>::type T;
    __shared__ int s_hist[256], s_slots[EV_NT / 64], s_pick[2];
    __shared__ int s_free[2 * EV_NT], s_from[2 * EV_NT];  // queues of free places and of movers
    const int tid = threadIdx.x, panel = blockIdx.x;
    const int per = a.b * a.h, layer = panel / per, sh = panel - layer * per, s = sh / a.h;
    const int cap = a.cap, n = (int)(a.ctx[s] < (uint32_t)cap ? a.ctx[s] : (uint32_t)cap);
    const size_t at = (size_t)(a.layer0 + layer) * per + sh;
    const uint64_t *mass = a.mass + at * cap;
    uint64_t *mass_out = a.mass_out + at * cap;
    uint32_t *kept = a.kept ? a.kept + at * a.budget : nullptr;
    if (a.ctx_out && at == (size_t)s * a.h && tid == 0) a.ctx_out[s] = (uint32_t)(n < a.budget ? n : a.budget);
    if (n <= a.budget) {
        for (int i = tid; i < n; i += EV_NT) {
            if (kept) kept[i] = i;
            if (mass != mass_out) mass_out[i] = mass[i];
        }
        return;
    }
    const int heavy = a.budget - a.recent, m = n - a.recent;  // m candidates, heavy < m
    // the heavy-th largest mass: `top` its value, `need` of the keys with exactly that value stay
    uint64_t top = 0;
    int need = heavy;
    for (int shift = 56; shift >= 0 && heavy > 0; shift -= 8) {
        s_hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < m; i += EV_NT) {
            const uint64_t x = mass[i];
            if (shift == 56 || (x >> (shift + 8)) == (top >> (shift + 8))) atomicAdd(&s_hist[(x >> shift) & 255], 1);
        }
        __syncthreads();
        // bin 255 - tid and the count above it
        int total;
        const int mine = s_hist[255 - tid], above = block_scan(mine, s_slots, tid, total);
        if (above < need && above + mine >= need) {
            s_pick[0] = 255 - tid;
            s_pick[1] = need - above;
        }
        __syncthreads();
        top |= (uint64_t)s_pick[0] << shift;
        need = s_pick[1];
    }
    int8_t *K = c.k[layer] + (size_t)sh * cap * a.hd, *V = c.v[layer] + (size_t)sh * cap * a.hd;
    const int words = a.hd / W, rows = EV_NT / words, r = tid / words, w = tid - r * words;
    int ties = 0;             // keys of value `top` before the scanned tile
    int n_free = 0, n_from = 0;
    int done = 0, src = heavy;  // the scans' next keys: [0, heavy) for free places, [heavy, m) for movers
    int ties_from = 0;        // keys of value `top` before src
    if (heavy > 0) {
        // the ties below `heavy`, so that the scan above it can run beside the one below
        int below = 0;
        for (int i = tid; i < heavy; i += EV_NT) below += mass[i] == top;
        int total;
        block_scan(below, s_slots, tid, total);
        ties_from = total;
    }
    auto member = [&](int i, int end, int &before) {
        const uint64_t x = i < end ? mass[i] : 0;
        const bool tie = i < end && x == top;
        int total;
        const int rank = before + block_scan(tie, s_slots, tid, total);
        before += total;
        return i < end && (x > top || (tie && rank < need));
    };
    while (heavy > 0) {
        while (n_free < EV_NT && done < heavy) {
            const int i = done + tid;
            const bool in = member(i, heavy, ties), free = i < heavy && !in;
            if (in) {
                if (kept) kept[i] = i;
                if (mass != mass_out) mass_out[i] = mass[i];
            }
            int total;
            const int rank = block_scan(free, s_slots, tid, total);
            if (free) s_free[n_free + rank] = i;
            n_free += total;
            done += EV_NT;
        }
        while (n_from < EV_NT && src < m) {
            const int i = src + tid;
            const bool in = member(i, m, ties_from);
            int total;
            const int rank = block_scan(in, s_slots, tid, total);
            if (in) s_from[n_from + rank] = i;
            n_from += total;
            src += EV_NT;
        }
        const int go = n_free < n_from ? n_free : n_from;  // 0 only when both are empty and scanned
        if (go == 0) break;
        __syncthreads();
        if (r < rows)
            for (int j = r; j < go; j += rows) {
                const size_t to = (size_t)s_free[j] * a.hd, from = (size_t)s_from[j] * a.hd;
                ((T *)(K + to))[w] = ((const T *)(K + from))[w];
                ((T *)(V + to))[w] = ((const T *)(V + from))[w];
            }
        for (int j = tid; j < go; j += EV_NT) {
            if (kept) kept[s_free[j]] = s_from[j];
            mass_out[s_free[j]] = mass[s_from[j]];
        }
        // the rest of the queues to their starts (at most EV_NT entries each)
        const int f = tid + go < n_free ? s_free[tid + go] : 0, q = tid + go < n_from ? s_from[tid + go] : 0;
        __syncthreads();
        if (tid + go < n_free) s_free[tid] = f;
        if (tid + go < n_from) s_from[tid] = q;
        n_free -= go;
        n_from -= go;
        __syncthreads();
    }
    __syncthreads();
    // the recent rows: m .. n - 1 to heavy .. budget - 1, a tile read whole before it is written
    const int8_t *K0 = K + (size_t)m * a.hd, *V0 = V + (size_t)m * a.hd;
    for (int j0 = 0; j0 < a.recent; j0 += rows) {
        const bool go = r < rows && j0 + r < a.recent;
        const size_t o = (size_t)(j0 + r) * a.hd;
        T kx, vx;
        if (go) {
            kx = ((const T *)(K0 + o))[w];
            vx = ((const T *)(V0 + o))[w];
        }
        __syncthreads();
        if (go) {
            ((T *)(K + (size_t)heavy * a.hd + o))[w] = kx;
            ((T *)(V + (size_t)heavy * a.hd + o))[w] = vx;
        }
        __syncthreads();
    }
    for (int j0 = 0; j0 < a.recent; j0 += EV_NT) {
        const int j = j0 + tid;
        const uint64_t x = j < a.recent ? mass[m + j] : 0;
        __syncthreads();
        if (j < a.recent) {
            mass_out[heavy + j] = x;
            if (kept) kept[heavy + j] = m + j;
        }
        __syncthreads();
    }
    for (int i = a.budget + tid; i < n; i += EV_NT) mass_out[i] = 0;
}

hipError_t launch_evict(const CachePtrs &c, int layers, const EvictArgs &a, hipStream_t stream) {
    const int panels = layers * a.b * a.h;
    if (panels <= 0) return hipSuccess;
    if (wide_words(c, layers, a.hd)) launch_k(k_evict<16>, dim3(panels), dim3(EV_NT), 0, stream, c, a);
    else launch_k(k_evict<4>, dim3(panels), dim3(EV_NT), 0, stream, c, a);
    return hipGetLastError();
}

}  // namespace hs
