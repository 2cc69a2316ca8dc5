// Caches in pages of a pool, 8 bits a value with a scale for each page and head (no counterpart in the reference, whose
// caches are one panel a slot with one static scale): appending rows, and attention over the pages.
#include "attend.h"

namespace hs {

// The scale of a page whose first row's largest magnitude is `most`: that row times headroom / 16 fits +-127.
__device__ __forceinline__ uint32_t page_scale(uint32_t most, const AppendArgs &a) {
    const uint32_t s = (most * a.headroom + 127 * 16 - 1) / (127 * 16);
    return s < 1 ? 1 : (s > a.pages.max_scale ? a.pages.max_scale : s);
}

// The stored byte of x: round(x / s), halves up, clamped.
__device__ __forceinline__ int8_t page_byte(int32_t x, int32_t s) {
    const int32_t n = 2 * x + s, d = 2 * s;
    int32_t q = n / d;
    if (n - q * d < 0) q--;
    return (int8_t)(q < -127 ? -127 : (q > 127 ? 127 : q));
}

__device__ __forceinline__ uint32_t held_scale(uint32_t s, uint32_t most) { return s < 1 ? 1 : (s > most ? most : s); }

// A wave for each (stream, row, head), K and V in turn.
template <typename X>
__global__ __launch_bounds__(256) void k_append(AppendArgs a, size_t n_tasks) {
    const int lane = threadIdx.x & 63;
    const size_t task = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (task >= n_tasks) return;
    const PagePool &p = a.pages;
    const int h = (int)(task % p.kv_heads), i = (int)(task / p.kv_heads % a.t), s = (int)(task / p.kv_heads / a.t);
    const uint32_t cap = (uint32_t)a.width * p.page, n = a.ctx[s] < cap ? a.ctx[s] : cap;
    uint32_t rows = a.rows ? a.rows[s] : (uint32_t)a.t;
    rows = rows < (uint32_t)a.t ? rows : (uint32_t)a.t;
    rows = rows < cap - n ? rows : cap - n;
    if (a.ctx_out && i == 0 && h == 0 && lane == 0) a.ctx_out[s] = n + rows;
    if ((uint32_t)i >= rows) return;
    const uint32_t at = n + i, place = at % p.page, number = a.table[(size_t)s * a.width + at / p.page];
    if (number >= (uint32_t)p.pages) return;
    const size_t panel = (size_t)number * p.kv_heads + h;
    for (int which = 0; which < 2; which++) {
        const X *x = (const X *)(which ? a.v : a.k) + ((size_t)s * a.t + i) * a.stride + (size_t)h * p.hd;
        int8_t *to = (which ? p.v : p.k) + (panel * p.page + place) * p.hd;
        uint32_t *scales = which ? p.v_scale : p.k_scale;
        uint32_t scale = 1;
        if (sizeof(X) > 1) {
            if (place <= (uint32_t)i) {  // the page's first row is of this call
                const X *first = x - (size_t)place * a.stride;
                int64_t most = 0;
                for (int c = lane; c < p.hd; c += 64) {
                    const int64_t m = first[c] < 0 ? -(int64_t)first[c] : first[c];
                    most = m > most ? m : most;
                }
                scale = page_scale((uint32_t)wave_max64(most), a);
            } else {
                scale = held_scale(scales[panel], p.max_scale);
            }
        }
        if (place == 0 && lane == 0) scales[panel] = scale;
        for (int c = lane; c < p.hd; c += 64) to[c] = sizeof(X) > 1 ? page_byte(x[c], (int32_t)scale) : (int8_t)x[c];
    }
}

hipError_t launch_append(const AppendArgs &a, hipStream_t stream) {
    const size_t tasks = (size_t)a.streams * a.t * a.pages.kv_heads;
    if (tasks == 0) return hipSuccess;
    const dim3 grid((unsigned)((tasks + 3) / 4));
    if (a.bits == 8) launch_k(k_append<int8_t>, grid, dim3(256), 0, stream, a, tasks);
    else launch_k(k_append<int16_t>, grid, dim3(256), 0, stream, a, tasks);
    return hipGetLastError();
}

// ---- Attention over the pages ------------------------------------------------------------------------
// score_j = clamp(rescale(q k_j, score_m ks, score_s), +-2^40), e_j = table[min(M - score_j, len - 1)], S = sum e_j,
// w_j = floor(e_j vs 2^P / S), out = clamp(rescale(sum w_j v_j, out_m, out_s), +-127), with ks and vs the scales of key
// j's page: the rule of the other attention kernels where the scales are 1.

struct PagedRows {
    int keys, rows;  // of the stream: row i sees keys 0 .. keys - rows + i
};
__device__ __forceinline__ PagedRows paged_rows(const PagedArgs &g, int s) {
    PagedRows r;
    r.keys = (int)(g.ctx[s] < (uint32_t)g.keys ? g.ctx[s] : (uint32_t)g.keys);
    const uint32_t n = g.rows ? g.rows[s] : (uint32_t)g.t;
    r.rows = (int)(n < (uint32_t)g.t ? n : (uint32_t)g.t);
    return r;
}

// A wave for each (row, head): three passes over the keys.
__global__ __launch_bounds__(256) void k_paged_rows(PagedArgs g, size_t n_tasks) {
    __shared__ __attribute__((aligned(16))) int s_q[4][64];
    const PagePool &p = g.pages;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = p.hd;
    const size_t task = (size_t)blockIdx.x * 4 + wave;
    const size_t row = task < n_tasks ? task / g.heads : 0;
    const int h = task < n_tasks ? (int)(task % g.heads) : 0;
    const int s = (int)(row / g.t), i = (int)(row % g.t);
    const PagedRows R = paged_rows(g, s);
    const bool live = task < n_tasks && i < R.rows;
    if (live && lane < hd / 4) s_q[wave][lane] = ((const int *)(g.q + row * g.q_stride + (size_t)h * hd))[lane];
    __syncthreads();
    if (!live) return;
    const int *q4 = s_q[wave];
    const int kvh = h / (g.heads / p.kv_heads), keys = R.keys - R.rows + i + 1;
    const int64_t last = g.exp_len - 1;
    const uint32_t *table = g.table + (size_t)s * g.width;
    struct Key {
        bool seen;
        size_t at;  // of its values
        uint32_t ks, vs;
    };
    auto find = [&](int j) {
        const uint32_t number = table[j / p.page];
        Key k;
        k.seen = number < (uint32_t)p.pages;
        const size_t panel = (size_t)(k.seen ? number : 0) * p.kv_heads + kvh;
        k.at = (panel * p.page + j % p.page) * hd;
        k.ks = held_scale(p.k_scale[panel], p.max_scale);
        k.vs = held_scale(p.v_scale[panel], p.max_scale);
        return k;
    };
    const int se = g.score_s < 63 ? g.score_s : 63;
    const int64_t half = se ? (int64_t)1 << (se - 1) : 0;
    auto score = [&](const Key &k) {
        const int64_t x = (int64_t)dot_key(q4, p.k + k.at, hd) * (int32_t)(g.score_m * k.ks);
        return clamp64((x + half) >> se, -SCORE_LIMIT, SCORE_LIMIT);
    };
    int64_t mx = INT64_MIN;
    for (int j = lane; j < keys; j += 64) {
        const Key k = find(j);
        const int64_t x = k.seen ? score(k) : INT64_MIN;
        mx = x > mx ? x : mx;
    }
    mx = wave_max64(mx);
    int64_t sum = 0;
    for (int j = lane; j < keys; j += 64) {
        const Key k = find(j);
        if (!k.seen) continue;
        const int64_t dd = mx - score(k);
        sum += g.exp_table[dd < last ? dd : last];
    }
    sum = wave_sum64(sum);
    int64_t acc[4] = {0, 0, 0, 0};
    for (int j0 = 0; j0 < keys && sum > 0; j0 += 64) {
        const int j = j0 + lane;
        int64_t w = 0, at = 0;
        if (j < keys) {
            const Key k = find(j);
            at = (int64_t)k.at;
            if (k.seen) {
                const int64_t dd = mx - score(k);
                w = (int64_t)((((uint64_t)(uint32_t)g.exp_table[dd < last ? dd : last] * k.vs) << g.softmax_p) / (uint64_t)sum);
            }
        }
        const int cnt = keys - j0 < 64 ? keys - j0 : 64;
        for (int jj = 0; jj < cnt; jj++) {
            const int64_t wj = __shfl(w, jj, 64);
            const int8_t *v = p.v + __shfl(at, jj, 64);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 64 * u < hd) acc[u] += wj * (int64_t)v[lane + 64 * u];
        }
    }
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < hd)
            g.out[(row * g.heads + h) * hd + lane + 64 * u] = (int8_t)clamp128(rescale_full(acc[u], g.out_m, g.out_s), -127, 127);
}

size_t paged_workspace(const PagedArgs &) { return 0; }

hipError_t launch_paged(const PagedArgs &g, void *, hipStream_t stream) {
    const size_t tasks = (size_t)g.streams * g.t * g.heads;
    if (tasks == 0) return hipSuccess;
    launch_k(k_paged_rows, dim3((unsigned)((tasks + 3) / 4)), dim3(256), 0, stream, g, tasks);
    return hipGetLastError();
}

}  // namespace hs
