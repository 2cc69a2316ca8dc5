// Appending rows to caches in pages of a pool, 8 bits a value with a scale for each page and head (no counterpart in the
// reference, whose caches are one panel a slot with one static scale).
#include "attend.h"

namespace hs {

// The scale of a page whose first row's largest magnitude is `most`: that row times headroom / 16 fits +-127.
__device__ __forceinline__ uint32_t page_scale(uint32_t most, const AppendArgs &a) {
    const uint32_t s = (most * a.headroom + 127 * 16 - 1) / (127 * 16);
    return s < 1 ? 1 : (s > a.pages.max_scale ? a.pages.max_scale : s);
}

// floor((2 x + s) / (2 s)) = floor(x / s + 1/2), clamped to +-127, in single precision: x / s + 1/2 is a multiple of 1 / (2 s), s <=
// 2^10, so it lies on an integer or 2^-11 from one; where the clamp does not decide, |x / s| < 128 and the roundings (1 / s, the
// multiply-add) are below 2^-15. 2^-13 added keeps them from reaching below an integer.
__device__ __forceinline__ int32_t page_byte(int32_t x, float inv) {
    return (int32_t)__builtin_amdgcn_fmed3f(floorf(fmaf((float)x, inv, 0.5f + 0x1p-13f)), -127.0f, 127.0f);
}

// A wave for each head of a run of tokens of one stream: CR tokens of one page (a run never crosses pages), K or V. A lane takes
// 16 channels of a row: 16 bytes of the page, so that a wave stores a whole KiB of it at a time, and reads 16 (i8) or 32
// (i16) bytes. Every wave takes the scale from the page's first row by itself, so no wave waits for another.
// HBM bounds it, two bytes read for one written: 64 streams x 1,024 tokens x 12 heads, 226 MB in 49 us, 4.6 TB/s (runs of whole pages
// of 64; what a wave finds out first is then one table entry and one row of 64). One token of 64 streams takes 5 us, a chain of
// the count, the page's number, its scale and the row, behind a call of 11 us on the host.
template <typename X>
__global__ __launch_bounds__(256) void k_append(AppendArgs a, int run, int runs, size_t n_tasks) {
    const PagePool &p = a.pages;
    const int lane = threadIdx.x & 63;
    const size_t task = (size_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (task >= n_tasks) return;
    const int which = (int)(task & 1), h = (int)((task >> 1) % p.kv_heads);
    const size_t rest = (task >> 1) / p.kv_heads;
    const int c = (int)(rest % runs), s = (int)(rest / runs);
    const uint32_t cap = (uint32_t)a.width * p.page, n = a.ctx[s] < cap ? a.ctx[s] : cap;
    uint32_t rows = a.rows ? a.rows[s] : (uint32_t)a.t;
    rows = rows < (uint32_t)a.t ? rows : (uint32_t)a.t;
    rows = rows < cap - n ? rows : cap - n;
    if (a.ctx_out && c == 0 && h == 0 && which == 0 && lane == 0) a.ctx_out[s] = n + rows;
    // the run's tokens t0 .. t1 - 1 of the stream's
    const uint32_t r0 = (n / run + c) * run, t0 = r0 > n ? r0 : n, t1 = r0 + run < n + rows ? r0 + run : n + rows;
    if (t0 >= t1) return;
    const uint32_t number = a.table[(size_t)s * a.width + t0 / p.page], start = t0 / p.page * p.page;
    if (number >= (uint32_t)p.pages) return;
    const size_t panel = (size_t)number * p.kv_heads + h;
    const X *from = (const X *)(which ? a.v : a.k) + (size_t)s * a.t * a.stride + (size_t)h * p.hd;  // token n
    int8_t *to = (which ? p.v : p.k) + (panel * p.page + t0 - start) * p.hd;
    uint32_t *scales = which ? p.v_scale : p.k_scale;
    const int units = p.hd / 16;  // of a row
    float inv = 1.0f;
    if constexpr (sizeof(X) > 1) {
        uint32_t scale;
        if (start >= n) {  // the page's first row is of this call
            int32_t most = 0;
            if (lane < units) {
                const v4i *x = (const v4i *)(from + (size_t)(start - n) * a.stride + 16 * lane);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const v4i y = x[k];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int32_t lo = (int16_t)y[e], hi = y[e] >> 16;
                        const int32_t al = lo < 0 ? -lo : lo, ah = hi < 0 ? -hi : hi;
                        most = al > most ? al : most;
                        most = ah > most ? ah : most;
                    }
                }
            }
            int32_t least = 0;
            wave_min_max(least, most);
            scale = page_scale((uint32_t)most, a);
            if (t0 == start && lane == 0) scales[panel] = scale;
        } else {
            scale = scales[panel];
            scale = scale < 1 ? 1 : (scale > p.max_scale ? p.max_scale : scale);
        }
        inv = 1.0f / (float)scale;
    } else if (t0 == start && lane == 0) {
        scales[panel] = 1;
    }
    const int total = (int)(t1 - t0) * units;
    for (int i0 = lane; i0 < total; i0 += 256) {
        constexpr int L = sizeof(X);  // 16-byte loads of a unit
        v4i x[4][L];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = i0 + 64 * k < total ? i0 + 64 * k : i0, row = i / units;
            const v4i *y = (const v4i *)(from + (size_t)(t0 - n + row) * a.stride + 16 * (i - row * units));
#pragma unroll
            for (int l = 0; l < L; l++) x[k][l] = y[l];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (i0 + 64 * k >= total) break;
            v4i out;
            if constexpr (sizeof(X) > 1) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int32_t lo = x[k][e >> 1][2 * (e & 1)], hi = x[k][e >> 1][2 * (e & 1) + 1];
                    const uint32_t b0 = page_byte((int16_t)lo, inv), b1 = page_byte(lo >> 16, inv), b2 = page_byte((int16_t)hi, inv),
                                   b3 = page_byte(hi >> 16, inv);
                    out[e] = (int32_t)((b0 & 255) | (b1 & 255) << 8 | (b2 & 255) << 16 | b3 << 24);
                }
            } else {
                out = x[k][0];
            }
            ((v4i *)to)[i0 + 64 * k] = out;
        }
    }
}

// Runs of up to 64 tokens: the most that t tokens of a stream touch.
static int append_run(const AppendArgs &a) { return a.pages.page < 64 ? a.pages.page : 64; }
static int append_runs(const AppendArgs &a) { return (a.t + 2 * append_run(a) - 2) / append_run(a); }

bool append_fits(const AppendArgs &a) {  // a wave a task, a grid of fewer than 2^32 threads
    return (size_t)a.streams * append_runs(a) * a.pages.kv_heads * 2 < ((size_t)1 << 26) - 4;
}

hipError_t launch_append(const AppendArgs &a, hipStream_t stream) {
    const int run = append_run(a), runs = append_runs(a);
    const size_t tasks = (size_t)a.streams * runs * a.pages.kv_heads * 2;
    const dim3 grid((unsigned)((tasks + 3) / 4));
    if (a.bits == 8) launch_k(k_append<int8_t>, grid, dim3(256), 0, stream, a, run, runs, tasks);
    else launch_k(k_append<int16_t>, grid, dim3(256), 0, stream, a, run, runs, tasks);
    return hipGetLastError();
}

}  // namespace hs
