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
// row is read before anything is written over it. A wave takes CM panels (K or V of a layer) of one (stream,
// head): what bounds it is the chain of loads (counts, path, rows), paid once for all of them, with
// their rows in flight together. (24 layers x 64 streams x 16 heads, 4 rows in the mean: 14.0 us a call with one panel a wave, 9.4 with eight.)
constexpr int CM = 8;

template <int W>
__global__ __launch_bounds__(256) void k_commit(CachePtrs c, CommitArgs a, int layers, int n_tasks) {
    typedef typename Word<W>::type T;
    const int lane = threadIdx.x & 63, task = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (task >= n_tasks) return;
    const int per = a.b * a.h, part = task / per, sh = task - part * per, s = sh / a.h;
    const uint32_t cap = (uint32_t)a.cap;
    const uint32_t ctx = a.ctx[s] < cap ? a.ctx[s] : cap;
    uint32_t acc = a.accepted[s] < (uint32_t)a.t ? a.accepted[s] : (uint32_t)a.t;
    acc = acc < cap - ctx ? acc : cap - ctx;
    if (a.ctx_out && part == 0 && a.first && sh == s * a.h && lane == 0) a.ctx_out[s] = ctx + acc;
    const int words = a.hd / W, rows = 64 / words, r = lane / words, w = lane - r * words;
    if (r >= rows) return;
    const size_t base = ((size_t)sh * cap + ctx) * a.hd;
    for (uint32_t i = r; i < acc; i += rows) {
        const uint32_t p = a.path[(size_t)s * a.t + i];
        if (p == i || p >= cap - ctx) continue;  // in place already; a row past the cache is left alone
        T x[CM];
#pragma unroll
        for (int u = 0; u < CM; u++) {
            const int panel = CM * part + u;  // K and V of a layer in turn
            if (panel < 2 * layers)
                x[u] = ((const T *)((panel & 1 ? c.v : c.k)[panel >> 1] + base + (size_t)p * a.hd))[w];
        }
#pragma unroll
        for (int u = 0; u < CM; u++) {
            const int panel = CM * part + u;
            if (panel < 2 * layers) ((T *)((panel & 1 ? c.v : c.k)[panel >> 1] + base + (size_t)i * a.hd))[w] = x[u];
        }
    }
}

static bool wide_words(const CachePtrs &c, int layers, int hd) {
    uintptr_t bits = (uintptr_t)hd;
    for (int l = 0; l < layers; l++) bits |= (uintptr_t)c.k[l] | (uintptr_t)c.v[l];
    return bits % 16 == 0;
}

hipError_t launch_commit(const CachePtrs &c, int layers, const CommitArgs &a, hipStream_t stream) {
    const int tasks = (2 * layers + CM - 1) / CM * a.b * a.h;
    if (tasks <= 0) return hipSuccess;
    const dim3 grid((tasks + 3) / 4);
    if (wide_words(c, layers, a.hd)) launch_k(k_commit<16>, grid, dim3(256), 0, stream, c, a, layers, tasks);
    else launch_k(k_commit<4>, grid, dim3(256), 0, stream, c, a, layers, tasks);
    return hipGetLastError();
}

// ---- evict -----------------------------------------------------------------------------------------
// One workgroup per (layer, stream, head) panel of n > budget keys. The `heavy` = budget - recent largest
// masses of the first n - recent keys stay (ties: the lowest index), by a radix selection of the
// heavy-th largest value, eight bits at a time. Attention over integers does not depend on the order of the
// keys, so only what must move moves: a kept key below `heavy` stays where it is, and the a-th free place below it
// takes the a-th kept key from above; the recent rows follow in order. Sources of the first kind lie at or above
// `heavy` and places below, so these copies need no order; the recent rows move down tile by tile after them.
// (k_evict: caches of more than 16,384 places. It walks the masses up to eight times for the selection and twice
// after it, 256 threads a panel: 256 panels of 32,768 places to 8,192 keys 635 us (531 MB: 111 at the rate of a copy), of
// 65,536 to 16,384 1,294; 12 panels 400 and 830.)

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

// Up to NT R keys a panel: a thread holds R masses, and everything follows from registers in a few barriers. A
// wave owns 64 R keys in a row, so the ranks of ties, free places and movers are wave ballots and one exchange of
// the waves' counts. The first digit of the selection is a mass's bit length and the four bits below the leading one
// (1,040 bins in the order of the values): accumulated weights spread over orders of magnitude, so a bin
// holds few of them, where the leading byte would hold almost all; then eight bits at a time among
// that bin's keys, until the rest of a bin stays whole.
// Copies of the kernel without a part: 9,216 panels of 1,024 places to 768 keys 107 us (375 MB), 27 without the copies of
// rows and masses, 35 with the masses alone; 256 panels of 16,384 to 4,096 103 us (274 MB), 24 and 31. So the rows' copies
// (half lines of 64 bytes) take 70% and start after the selection: one workgroup fills a CU at 16,384 places, and nothing
// moves rows while it selects. That is no limit: the recent rows could be in flight by then.
constexpr int EV_BINS = 1040;

__device__ __forceinline__ int mass_bin(uint64_t x) {
    if (x == 0) return 0;
    const int e = 63 - __builtin_clzll(x);
    const int m = (int)(e >= 4 ? x >> (e - 4) : x << (4 - e)) & 15;
    return 16 * (e + 1) + m;
}

// s_hist[bin] += 1 for the lanes with `on`; one addition where the whole wave has the same bin.
__device__ __forceinline__ void count_bin(int *s_hist, int bin, bool on) {
    const uint64_t lanes = __ballot(on);
    if (lanes == 0) return;
    const int lead = __builtin_ctzll(lanes), first = __shfl(bin, lead, 64);
    if (__ballot(on && bin == first) == lanes) {
        if ((int)(threadIdx.x & 63) == lead) atomicAdd(&s_hist[first], __popcll(lanes));
    } else if (on) {
        atomicAdd(&s_hist[bin], 1);
    }
}

// The sum of v over the workgroup's threads before this one; `slots` holds a value per wave.
template <int NT>
__device__ __forceinline__ int scan_threads(int v, int *slots, int lane, int w) {
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) slots[w] = x;
    __syncthreads();
    int before = x - v;
    for (int i = 0; i < w; i++) before += slots[i];
    return before;
}

template <int W, int NT, int R>
__global__ __launch_bounds__(NT) void k_evict_regs(CachePtrs c, EvictArgs a) {
    typedef typename Word<W>::type T;
    constexpr int NW = NT / 64, BPT = (EV_BINS + NT - 1) / NT;
    extern __shared__ uint32_t s_list[];  // NT R / 2 free places, then as many movers
    __shared__ int s_hist[BPT * NT], s_slots[2][NW], s_pick[3];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), panel = blockIdx.x;
    const int per = a.b * a.h, layer = panel / per, sh = panel - layer * per, s = sh / a.h;
    const int cap = a.cap, n = (int)(a.ctx[s] < (uint32_t)cap ? a.ctx[s] : (uint32_t)cap);
    const size_t at = (size_t)(a.layer0 + layer) * per + sh;
    const uint64_t *mass = a.mass + at * cap;
    uint64_t *mass_out = a.mass_out + at * cap;
    uint32_t *kept = a.kept ? a.kept + at * a.budget : nullptr;
    if (a.ctx_out && at == (size_t)s * a.h && tid == 0) a.ctx_out[s] = (uint32_t)(n < a.budget ? n : a.budget);
    const int i0 = 64 * R * w + lane;  // the thread's keys: i0 + 64 j
    uint64_t x[R];
#pragma unroll
    for (int j = 0; j < R; j++) x[j] = i0 + 64 * j < n ? mass[i0 + 64 * j] : 0;
    if (n <= a.budget) {
#pragma unroll
        for (int j = 0; j < R; j++)
            if (i0 + 64 * j < n) {
                if (kept) kept[i0 + 64 * j] = i0 + 64 * j;
                if (mass != mass_out) mass_out[i0 + 64 * j] = x[j];
            }
        return;
    }
    const int heavy = a.budget - a.recent, m = n - a.recent;
    // Of the first m keys stay those with x >> sh > pre, and the first `need` of those where they are equal.
    uint64_t pre = ~(uint64_t)0;
    int shift = 0, need = heavy, size = 0;  // size: the keys where they are equal
    if (heavy > 0) {
        // the bin (from the last one down) in which the need-th key from above lies
        auto pick = [&](int bins_a_thread) {
            int mine = 0;
            for (int b = 0; b < bins_a_thread; b++) mine += s_hist[bins_a_thread * NT - 1 - (bins_a_thread * tid + b)];
            int above = scan_threads<NT>(mine, s_slots[0], lane, w);
            if (above < need && above + mine >= need) {
                int b = bins_a_thread * NT - 1 - bins_a_thread * tid;
                while (above + s_hist[b] < need) above += s_hist[b--];
                s_pick[0] = b;
                s_pick[1] = need - above;
                s_pick[2] = s_hist[b];
            }
            __syncthreads();
            need = s_pick[1];
            size = s_pick[2];
            return s_pick[0];
        };
        for (int b = tid; b < BPT * NT; b += NT) s_hist[b] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < R; j++)
            if (64 * (R * w + j) < m) count_bin(s_hist, mass_bin(x[j]), i0 + 64 * j < m);
        __syncthreads();
        const int bin = pick(BPT);
        const int e = bin / 16 - 1;  // the bit length less one; -1: zeros
        if (e < 0) pre = 0;
        else if (e < 4) pre = (uint64_t)(16 + bin % 16) >> (4 - e);
        else pre = 16 + bin % 16, shift = e - 4;
        while (shift > 0 && size > need) {
            const int next = shift > 8 ? shift - 8 : 0, mask = (1 << (shift - next)) - 1;
            __syncthreads();  // (everyone has read the picked bin)
            for (int b = tid; b < (NT < 256 ? 256 : NT); b += NT) s_hist[b] = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < R; j++)
                if (64 * (R * w + j) < m) count_bin(s_hist, (int)(x[j] >> next) & mask, i0 + 64 * j < m && x[j] >> shift == pre);
            __syncthreads();
            const int digit = pick(1);
            pre = pre << (shift - next) | (uint64_t)digit;
            shift = next;
        }
    }
    // who stays; ties in order, where not all of them do
    uint32_t in = 0;
    {
        int ties = 0;
        uint64_t t[R];
#pragma unroll
        for (int j = 0; j < R; j++) {
            t[j] = __ballot(i0 + 64 * j < m && heavy > 0 && x[j] >> shift == pre);
            ties += __popcll(t[j]);
        }
        if (lane == 0) s_slots[1][w] = ties;
        __syncthreads();
        int rank = 0;
        for (int i = 0; i < w; i++) rank += s_slots[1][i];
#pragma unroll
        for (int j = 0; j < R; j++) {
            const int mine = rank + __builtin_amdgcn_mbcnt_hi((uint32_t)(t[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)t[j], 0));
            const bool tie = (t[j] >> lane) & 1;
            if (i0 + 64 * j < m && heavy > 0 && (x[j] >> shift > pre || (tie && mine < need))) in |= 1u << j;
            rank += __popcll(t[j]);
        }
    }
    uint32_t *s_free = s_list, *s_from = s_list + NT * R / 2;
    int moves;
    uint32_t from_rank[R];
    {
        int f = 0, q = 0;
        uint64_t bf[R], bq[R];
#pragma unroll
        for (int j = 0; j < R; j++) {
            const bool stay = (in >> j) & 1;
            bf[j] = __ballot(i0 + 64 * j < heavy && !stay);
            bq[j] = __ballot(i0 + 64 * j >= heavy && stay);
            f += __popcll(bf[j]);
            q += __popcll(bq[j]);
        }
        __syncthreads();
        if (lane == 0) {
            s_slots[0][w] = f;
            s_slots[1][w] = q;
        }
        __syncthreads();
        int fr = 0, qr = 0;
        moves = 0;
        for (int i = 0; i < NW; i++) {
            fr += i < w ? s_slots[0][i] : 0;
            qr += i < w ? s_slots[1][i] : 0;
            moves += s_slots[1][i];
        }
#pragma unroll
        for (int j = 0; j < R; j++) {
            if ((bf[j] >> lane) & 1)
                s_free[fr + __builtin_amdgcn_mbcnt_hi((uint32_t)(bf[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bf[j], 0))] = i0 + 64 * j;
            from_rank[j] = qr + __builtin_amdgcn_mbcnt_hi((uint32_t)(bq[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bq[j], 0));
            if ((bq[j] >> lane) & 1) s_from[from_rank[j]] = i0 + 64 * j;
            fr += __popcll(bf[j]);
            qr += __popcll(bq[j]);
        }
    }
    __syncthreads();  // the lists; and every mass has been read
    int8_t *K = c.k[layer] + (size_t)sh * cap * a.hd, *V = c.v[layer] + (size_t)sh * cap * a.hd;
    const int words = a.hd / W, rows = NT / words, r = tid / words, wd = tid - r * words;
    constexpr int U = 2;  // rows a thread has in flight, K and V of each
    if (r < rows)
        for (int j = r; j < moves; j += U * rows) {
            T kx[U], vx[U];
            uint32_t to[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int q = j + u * rows < moves ? j + u * rows : j;
                to[u] = s_free[q];
                const size_t o = (size_t)s_from[q] * a.hd;
                kx[u] = ((const T *)(K + o))[wd];
                vx[u] = ((const T *)(V + o))[wd];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (j + u * rows >= moves) break;
                const size_t o = (size_t)to[u] * a.hd;
                ((T *)(K + o))[wd] = kx[u];
                ((T *)(V + o))[wd] = vx[u];
            }
        }
#pragma unroll
    for (int j = 0; j < R; j++) {
        const int i = i0 + 64 * j;
        if (i >= n) continue;
        int to = i;  // the key's place, if it has one
        if (i >= m) to = heavy + (i - m);
        else if (!((in >> j) & 1)) to = -1;
        else if (i >= heavy) to = (int)s_free[from_rank[j]];
        if (to >= 0) {
            mass_out[to] = x[j];
            if (kept) kept[to] = i;
        }
        if (i >= a.budget) mass_out[i] = 0;
    }
    // the recent rows: m .. n - 1 to heavy .. budget - 1, a tile read whole before it is written
    const int8_t *K0 = K + (size_t)m * a.hd, *V0 = V + (size_t)m * a.hd;
    K += (size_t)heavy * a.hd;
    V += (size_t)heavy * a.hd;
    for (int j0 = 0; j0 < a.recent; j0 += U * rows) {
        T kx[U], vx[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = j0 + u * rows + r;
            if (r < rows && j < a.recent) {
                kx[u] = ((const T *)(K0 + (size_t)j * a.hd))[wd];
                vx[u] = ((const T *)(V0 + (size_t)j * a.hd))[wd];
            }
        }
        __syncthreads();  // (the first one: the movers have been read, too)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = j0 + u * rows + r;
            if (r < rows && j < a.recent) {
                ((T *)(K + (size_t)j * a.hd))[wd] = kx[u];
                ((T *)(V + (size_t)j * a.hd))[wd] = vx[u];
            }
        }
        __syncthreads();
    }
}

template <int W>
static hipError_t launch_evict_w(const CachePtrs &c, int panels, const EvictArgs &a, hipStream_t stream) {
    auto run = [&](auto kernel, int nt, int r) {
        const size_t lds = (size_t)4 * nt * r;
        const hipError_t e = allow_dynamic_lds((const void *)kernel, lds);
        if (e != hipSuccess) return e;
        launch_k(kernel, dim3(panels), dim3(nt), lds, stream, c, a);
        return hipGetLastError();
    };
    if (a.cap <= 1024) return run(k_evict_regs<W, 256, 4>, 256, 4);
    if (a.cap <= 4096) return run(k_evict_regs<W, 512, 8>, 512, 8);
    if (a.cap <= 16384) return run(k_evict_regs<W, 1024, 16>, 1024, 16);
    launch_k(k_evict<W>, dim3(panels), dim3(EV_NT), 0, stream, c, a);
    return hipGetLastError();
}

hipError_t launch_evict(const CachePtrs &c, int layers, const EvictArgs &a, hipStream_t stream) {
    const int panels = layers * a.b * a.h;
    if (panels <= 0) return hipSuccess;
    return wide_words(c, layers, a.hd) ? launch_evict_w<16>(c, panels, a, stream) : launch_evict_w<4>(c, panels, a, stream);
}

}  // namespace hs
