// Appending rows to caches in pages of a pool, 8 bits a value with a scale for each page and head (no counterpart in the
// reference, whose caches are one panel a slot with one static scale).
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

}  // namespace hs
