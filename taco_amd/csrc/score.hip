// Scores of rows of logits (no counterpart in the reference, whose callers get the weights of a whole row): the log
// probability and the rank of a given token, the entropy, and the first alternatives with their log probabilities.
// With M the row's largest logit, d = min(M - l, len - 1) a symbol's table index (logits.rs:62-72), w = table[d] and
// T = sum w: the log probability of a symbol is ln(w / T), the entropy sum (w / T) ln(T / w), and the symbols' order is
// by (d, symbol). M, d, w, T, ranks and the order are integers; only the logarithms round.
#include "attend.h"

namespace hs {

// ln(w / T) for w <= T: T - w is exact, so that a probability close to 1 keeps its digits.
__device__ __forceinline__ double log_share(uint64_t w, uint64_t total) {
    return w ? -log1p((double)(total - w) / (double)w) : -(double)INFINITY;
}

// A row of logits: the largest, and the table index of a symbol.
template <int SRC>
struct ScoreRow {
    const ScoreArgs &a;
    size_t row;
    int last;
    __device__ __forceinline__ ScoreRow(const ScoreArgs &args, int r) : a(args), row(r), last(args.table_len - 1) {}
    __device__ __forceinline__ int64_t value(int j) const {
        if constexpr (SRC == SCORE_I32) return ((const int32_t *)a.logits)[row * a.ld + j];
        else return ((const int64_t *)a.logits)[row * a.ld + j];
    }
    // what the row max is the largest of
    __device__ __forceinline__ int maxima() const { return SRC == SCORE_COMPACT ? a.ntiles : a.vocab; }
    __device__ __forceinline__ int64_t maximum(int j) const {
        if constexpr (SRC == SCORE_COMPACT) return a.tmax[row * a.ntiles + j];
        else return value(j);
    }
    __device__ __forceinline__ int index(int64_t M, int j) const {
        uint64_t d;  // (unsigned: exact for any two logits)
        if constexpr (SRC == SCORE_COMPACT) d = (uint64_t)M - (uint64_t)a.tmax[row * a.ntiles + (j >> 6)] + a.d16[row * a.ld16 + j];
        else d = (uint64_t)M - (uint64_t)value(j);
        return d < (uint64_t)last ? (int)d : last;
    }
};

// Any vocabulary and table: a workgroup a row, which walks it for the row max, the sum, the entropy and the rank, and
// once for each alternative (the next in the order after the one before).
template <int SRC>
__global__ __launch_bounds__(256) void k_score_any(ScoreArgs a) {
    __shared__ uint64_t s_u[4];
    __shared__ double s_d[4];
    const int tid = threadIdx.x, r = blockIdx.x, V = a.vocab;
    const ScoreRow<SRC> row(a, r);
    auto all = [&](auto v, auto *slots, auto join) {  // join over the workgroup
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o, 64));
        __syncthreads();
        if ((tid & 63) == 0) slots[tid >> 6] = v;
        __syncthreads();
        return join(join(slots[0], slots[1]), join(slots[2], slots[3]));
    };
    int64_t mx = INT64_MIN;
    for (int j = tid; j < row.maxima(); j += 256) {
        const int64_t x = row.maximum(j);
        mx = x > mx ? x : mx;
    }
    const int64_t M = all(mx, (int64_t *)s_u, [](int64_t x, int64_t y) { return x > y ? x : y; });
    auto add = [](uint64_t x, uint64_t y) { return x + y; };
    const uint32_t token = a.tokens ? a.tokens[r] : 0xffffffffu;
    const int td = token < (uint32_t)V ? row.index(M, (int)token) : 0;
    uint64_t sum = 0, ahead = 0;
    for (int j = tid; j < V; j += 256) {
        const int d = row.index(M, j);
        sum += a.table[d];
        ahead += d < td || (d == td && (uint32_t)j < token);
    }
    const uint64_t T = all(sum, s_u, add);
    ahead = all(ahead, s_u, add);
    if (tid == 0) {
        const bool some = token < (uint32_t)V;
        if (a.logprob) a.logprob[r] = some ? (float)log_share(a.table[td], T) : 0.0f;
        if (a.rank) a.rank[r] = some ? (uint32_t)ahead : 0xffffffffu;
    }
    if (a.entropy) {
        double h = 0;
        for (int j = tid; j < V; j += 256) {
            const uint64_t w = a.table[row.index(M, j)];
            if (w) h -= (double)w / (double)T * log_share(w, T);
        }
        h = all(h, s_d, [](double x, double y) { return x + y; });
        if (tid == 0) a.entropy[r] = (float)h;
    }
    int64_t before = -1;  // (d, symbol) of the last one found
    for (int i = 0; i < a.top; i++) {
        int64_t next = INT64_MAX;
        for (int j = tid; j < V; j += 256) {
            const int64_t x = (int64_t)row.index(M, j) << 32 | j;
            if (x > before && x < next) next = x;
        }
        before = all(next, (int64_t *)s_u, [](int64_t x, int64_t y) { return x < y ? x : y; });
        if (tid == 0) {
            if (a.top_tokens) a.top_tokens[(size_t)r * a.top + i] = (uint32_t)before;
            if (a.top_logprob) a.top_logprob[(size_t)r * a.top + i] = (float)log_share(a.table[before >> 32], T);
        }
    }
}

hipError_t launch_score(const ScoreArgs &a, int n_rows, hipStream_t stream) {
    if (n_rows <= 0) return hipSuccess;
    const dim3 grid(n_rows), block(256);
    if (a.src == SCORE_I32) launch_k(k_score_any<SCORE_I32>, grid, block, 0, stream, a);
    else if (a.src == SCORE_I64) launch_k(k_score_any<SCORE_I64>, grid, block, 0, stream, a);
    else launch_k(k_score_any<SCORE_COMPACT>, grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace hs
