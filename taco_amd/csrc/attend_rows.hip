// Integer attention of several query rows a stream (reference.rs:254-283, softmax.rs:78-104): the nodes of
// a tree of drafted tokens, each seeing the context and its ancestors, or a causal chunk of rows, with each
// key's weights p added to a 64-bit accumulator where the caller keeps one. No counterpart in the
// reference: it drafts chains, and its caches hold every key.
#include "attend.h"

namespace hs {

// The rows of one stream: row i is row first + i of q and out; it sees keys 0 .. full(i) - 1, and with a
// mask key base + n where bit n of its mask words is set (n < count).
struct StreamRows {
    int first, count, slot, base;
    const uint64_t *mask;  // the stream's first mask row
};

__device__ __forceinline__ StreamRows stream_rows(const RowsArgs &g, int s) {
    StreamRows R;
    if (g.groups) {
        const AttnGroup G = g.groups[s];
        R.first = G.first;
        R.count = G.count;
        R.slot = G.slot;
        R.base = G.pos0;
        R.mask = g.mask ? g.mask + (size_t)G.first * g.words : nullptr;
        return R;
    }
    const uint32_t cap = (uint32_t)g.a.ctx_cap, t = (uint32_t)g.t;
    uint32_t n = g.ctx[s] < cap ? g.ctx[s] : cap;  // never read past the cache
    uint32_t c = g.count ? g.count[s] : t;
    c = c < t ? c : t;
    R.first = s * g.t;
    R.slot = s;
    R.count = (int)c;
    R.base = g.mask ? (int)n : (int)n - (int)c;
    R.mask = g.mask ? g.mask + (size_t)R.first * g.words : nullptr;
    return R;
}

// One past the last key that any row of the stream sees.
__device__ __forceinline__ int stream_keys(const RowsArgs &g, const StreamRows &R) {
    const int n = R.base + R.count;
    return n < g.a.ctx_cap ? n : g.a.ctx_cap;
}

__device__ __forceinline__ bool row_sees(const RowsArgs &g, const StreamRows &R, int i, int key) {
    if (!g.mask) return key <= R.base + i;
    const int n = key - R.base;
    return n < 0 || ((R.mask[(size_t)i * g.words + (n >> 6)] >> (n & 63)) & 1) != 0;
}

// Any head dim that is a multiple of 4, any key count and table: one wave per (row, head), three passes over
// the keys as in k_attend (the row max, the sum of the entries, p and sum p v).
__global__ __launch_bounds__(256) void k_rows(RowsArgs g, int n_tasks) {
    __shared__ __attribute__((aligned(16))) int s_q[4][64];
    const AttnArgs &a = g.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int task = blockIdx.x * 4 + wave;
    const int row = task < n_tasks ? task / a.n_head : 0, h = task < n_tasks ? task % a.n_head : 0;
    const int s = row / g.t, i = row - s * g.t, hd = a.hd;
    const StreamRows R = stream_rows(g, s);
    const bool live = task < n_tasks && i < R.count;
    if (live && lane < hd / 4) s_q[wave][lane] = ((const int *)(a.q + (size_t)(R.first + i) * a.ldq + h * hd))[lane];
    __syncthreads();
    if (!live) return;
    const int *q4 = s_q[wave];
    const size_t panel = (size_t)R.slot * a.n_head + h;
    const int8_t *K = a.kc + panel * a.ctx_cap * hd, *V = a.vc + panel * a.ctx_cap * hd;
    const int keys = stream_keys(g, R);
    const int64_t last = a.exp_len - 1;
    auto score = [&](int j) { return attn_score<false>(a, dot_key(q4, K + (size_t)j * hd, hd)); };

    int64_t mx = INT64_MIN;
    for (int j = lane; j < keys; j += 64) {
        if (!row_sees(g, R, i, j)) continue;
        const int64_t x = score(j);
        mx = x > mx ? x : mx;
    }
    mx = wave_max64(mx);
    int64_t sum = 0;
    for (int j = lane; j < keys; j += 64) {
        if (!row_sees(g, R, i, j)) continue;
        const int64_t dd = mx - score(j);
        sum += a.exp_table[dd < last ? dd : last];
    }
    sum = wave_sum64(sum);
    int64_t acc[4] = {0, 0, 0, 0};
    for (int j0 = 0; j0 < keys && sum > 0; j0 += 64) {
        const int j = j0 + lane;
        uint64_t p = 0;
        if (j < keys && row_sees(g, R, i, j)) {
            const int64_t dd = mx - score(j);
            p = ((uint64_t)a.exp_table[dd < last ? dd : last] << a.softmax_p) / (uint64_t)sum;
            if (g.mass && p) atomicAdd((unsigned long long *)g.mass + panel * a.ctx_cap + j, (unsigned long long)p);
        }
        const int cnt = keys - j0 < 64 ? keys - j0 : 64;
        for (int jj = 0; jj < cnt; jj++) {
            const int64_t pj = (int64_t)__shfl(p, jj, 64);
            const int8_t *v = V + (size_t)(j0 + jj) * hd;
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (lane + 64 * u < hd) acc[u] += pj * (int64_t)v[lane + 64 * u];
        }
    }
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (lane + 64 * u < hd)
            *attn_out(a, R.first + i, h * hd + lane + 64 * u) =
                (int8_t)clamp128(rescale_full(acc[u], a.out_m, a.out_s), -127, 127);
}

size_t rows_workspace(const RowsArgs &) { return 0; }

hipError_t launch_rows(const RowsArgs &g, void *, hipStream_t stream) {
    const int tasks = g.streams * g.t * g.a.n_head;
    if (tasks <= 0) return hipSuccess;
    launch_k(k_rows, dim3((tasks + 3) / 4), dim3(256), 0, stream, g, tasks);
    return hipGetLastError();
}

}  // namespace hs
