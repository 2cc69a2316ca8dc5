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

// What a row's results need: the token's log probability and rank, and an alternative.
__device__ __forceinline__ void put_token(const ScoreArgs &a, size_t r, bool some, uint64_t w, uint64_t total, uint32_t rank) {
    if (a.logprob) a.logprob[r] = some ? (float)log_share(w, total) : 0.0f;
    if (a.rank) a.rank[r] = some ? rank : 0xffffffffu;
}
__device__ __forceinline__ void put_top(const ScoreArgs &a, size_t r, int i, uint32_t token, int d, uint64_t total) {
    if (a.top_tokens) a.top_tokens[r * a.top + i] = token;
    if (a.top_logprob) a.top_logprob[r * a.top + i] = (float)log_share(a.table[d], total);
}

// join over a workgroup of NW waves
template <int NW, typename T, typename F>
__device__ __forceinline__ T block_join(T v, void *slots, F join) {
    T *s = (T *)slots;
    const int tid = threadIdx.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((tid & 63) == 0) s[tid >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int i = 1; i < NW; i++) v = join(v, s[i]);
    return v;
}
struct Add {
    template <typename T>
    __device__ T operator()(T x, T y) const { return x + y; }
};
struct Max {
    template <typename T>
    __device__ T operator()(T x, T y) const { return x > y ? x : y; }
};
struct Min {
    template <typename T>
    __device__ T operator()(T x, T y) const { return x < y ? x : y; }
};

// The alternatives of a row, one walk each: the next in the order after the one before.
template <int SRC, int NW>
__device__ __forceinline__ void search_top(const ScoreArgs &a, size_t r, int64_t M, uint64_t T, void *slots) {
    const ScoreRow<SRC> row(a, r);
    int64_t before = -1;  // (d, symbol) of the last one found
    for (int i = 0; i < a.top; i++) {
        int64_t next = INT64_MAX;
        for (int j = threadIdx.x; j < a.vocab; j += 64 * NW) {
            const int64_t x = (int64_t)row.index(M, j) << 32 | j;
            if (x > before && x < next) next = x;
        }
        before = block_join<NW>(next, slots, Min());
        if (threadIdx.x == 0) put_top(a, r, i, (uint32_t)before, (int)(before >> 32), T);
    }
}

// A row by itself, any vocabulary and table: the workgroup walks it for the row max, the sum, the entropy and the rank,
// and for the alternatives.
template <int SRC, int NW>
__device__ __forceinline__ void score_any_row(const ScoreArgs &a, size_t r, void *slots) {
    const int tid = threadIdx.x, V = a.vocab, NT = 64 * NW;
    const ScoreRow<SRC> row(a, r);
    int64_t mx = INT64_MIN;
    for (int j = tid; j < row.maxima(); j += NT) {
        const int64_t x = row.maximum(j);
        mx = x > mx ? x : mx;
    }
    const int64_t M = block_join<NW>(mx, slots, Max());
    const uint32_t token = a.tokens ? a.tokens[r] : 0xffffffffu;
    const bool some = token < (uint32_t)V;
    const int td = some ? row.index(M, (int)token) : 0;
    uint64_t sum = 0, ahead = 0;
    for (int j = tid; j < V; j += NT) {
        const int d = row.index(M, j);
        sum += a.table[d];
        ahead += d < td || (d == td && (uint32_t)j < token);
    }
    const uint64_t T = block_join<NW>(sum, slots, Add());
    ahead = block_join<NW>(ahead, slots, Add());
    if (tid == 0) put_token(a, r, some, a.table[td], T, (uint32_t)ahead);
    if (a.entropy) {
        double h = 0;
        for (int j = tid; j < V; j += NT) {
            const uint64_t w = a.table[row.index(M, j)];
            if (w) h -= (double)w / (double)T * log_share(w, T);
        }
        h = block_join<NW>(h, slots, Add());
        if (tid == 0) a.entropy[r] = (float)h;
    }
    search_top<SRC, NW>(a, r, M, T, slots);
}
template <int SRC>
__global__ __launch_bounds__(512) void k_score_any(ScoreArgs a) {
    __shared__ uint64_t slots[8];
    score_any_row<SRC, 8>(a, blockIdx.x, slots);
}

// A row in the registers of a workgroup: read once, 4 G symbols a lane, their table indexes kept in 16 bits each and counted
// in an LDS histogram. Symbols past the table's end (and the places of the last groups past the row) go to 64 spare bins, each
// lane's in its own, so that no symbol needs a test and none of these many collide. The counts give T, the entropy and the
// token's rank but for ties; one wave walks them for the index up to which the alternatives lie, and the symbols up to
// there, few, are collected and ranked against each other.
constexpr int SCORE_LIST = 1024;   // symbols collected; where ties make them more, the alternatives are searched one by one
constexpr int SCORE_BINS = 16384;  // entries of the table at most

template <int SRC, int G, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(4))) void k_score_rows(ScoreArgs a) {
    constexpr int NT = 64 * NW;
    extern __shared__ uint32_t s_hist[];  // [table_len + 63]
    __shared__ uint64_t slots[NW], s_sum[NW], s_list[SCORE_LIST];
    __shared__ double s_ent[NW];
    __shared__ uint32_t s_ahead[NW], s_count, s_thr, s_found;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.vocab, last = a.table_len - 1;
    const size_t r = blockIdx.x;
    const uint32_t token = a.tokens ? a.tokens[r] : 0xffffffffu;
    const bool some = token < (uint32_t)V;
    const uint32_t cap = (uint32_t)(last + lane);  // this lane's bin of what lies past the table's end
    uint32_t d2[2 * G];                            // min(d, cap), pairs
    int off = 0;                                   // symbol of element e of group i: 4 (NT i + tid) + e - off
    int td = 0;                                    // the token's index
    int64_t top_logit;                             // the largest
    const ScoreRow<SRC> row(a, (int)r);
    auto symbol = [&](int i, int e) { return 4 * (NT * i + tid) + e - off; };
    auto inside = [&](int j) { return j >= 0 && j < V; };
    auto edge = [&](int i) { return (i == 0 && off > 0) || 4 * NT * (i + 1) > V + off; };  // some of group i are past the row (uniform)
    auto load = [](__amdgpu_buffer_rsrc_t x, int at, int step) { return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(x, at, step, 0)); };
    if (a.table[0] == 0) {  // (not a table of a model: the entropy below divides by it)
        score_any_row<SRC, NW>(a, r, slots);
        return;
    }
    for (int k = tid; k < last + 64; k += NT) s_hist[k] = 0;
    if (tid == 0) s_count = 0;

    if constexpr (SRC == SCORE_COMPACT) {
        const int64_t *tm = a.tmax + r * a.ntiles;
        const uint16_t *p = a.d16 + r * a.ld16;  // whole tiles of 64 (the row is padded)
        uint2 raw[G];
        int64_t t[G];
#pragma unroll
        for (int i = 0; i < G; i++) {
            const int j = symbol(i, 0) < V ? symbol(i, 0) : 0;
            raw[i] = *(const uint2 *)(p + j);
            t[i] = tm[j >> 6];
        }
        int64_t mx = INT64_MIN;
        for (int j = tid; j < a.ntiles; j += NT) mx = tm[j] > mx ? tm[j] : mx;
        const int64_t M = top_logit = block_join<NW>(mx, slots, Max());
        if (some) td = row.index(M, (int)token);
#pragma unroll
        for (int i = 0; i < G; i++) {
            const uint64_t b = (uint64_t)M - (uint64_t)t[i];
            const uint32_t base = b < (uint64_t)cap ? (uint32_t)b : cap;
            uint32_t d[4] = {raw[i].x & 0xffffu, raw[i].x >> 16, raw[i].y & 0xffffu, raw[i].y >> 16};
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = d[e] + base < (uint32_t)last ? d[e] + base : cap;  // (a d16 may be capped at last)
            d2[2 * i] = d[0] | d[1] << 16;
            d2[2 * i + 1] = d[2] | d[3] << 16;
        }
    } else {
        // 16-byte loads, from the 16 bytes that the row starts in to those that it ends in; zeros past them
        constexpr int E = SRC == SCORE_I32 ? 4 : 8;
        const uintptr_t at = (uintptr_t)a.logits + r * a.ld * E;
        off = (int)(at % 16) / E;
        const int bytes = ((off + V) * E + 15) / 16 * 16;
        const auto from = __builtin_amdgcn_make_buffer_rsrc((void *)(at - at % 16), 0, bytes, 0x00020000);
        const int64_t of_token = some ? row.value((int)token) : 0;
        // i32 logits as they are, i64 ones as their difference to 2^31 below the row's first one, in 32 bits
        typedef typename std::conditional<SRC == SCORE_I32, int32_t, uint32_t>::type X;
        constexpr X LOW = SRC == SCORE_I32 ? (X)INT32_MIN : (X)0;
        X x[4 * G], mx = LOW;
        uint64_t ref = 0;
        uint32_t apart = 0;  // not 0: they do not fit
        auto take = [&](int i) {
            if (edge(i)) {
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * i + e] = inside(symbol(i, e)) ? x[4 * i + e] : LOW;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) mx = x[4 * i + e] > mx ? x[4 * i + e] : mx;
        };
        if constexpr (SRC == SCORE_I32) {
#pragma unroll
            for (int i = 0; i < G; i++) {
                const uint4 y = load(from, 16 * tid, 16 * NT * i);
                x[4 * i] = (int32_t)y.x;
                x[4 * i + 1] = (int32_t)y.y;
                x[4 * i + 2] = (int32_t)y.z;
                x[4 * i + 3] = (int32_t)y.w;
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < G; i++) take(i);
        } else {
            const int64_t first = ((const int64_t *)at)[0];
            // (a first logit at the types' ends: the differences would come round)
            if (first >= (int64_t)1 << 62 || first < -((int64_t)1 << 62)) apart = 1;
            ref = (uint64_t)first - 0x80000000u;
            constexpr int B = 4;  // groups in flight beside those at work
            uint4 raw[2][B][2];
            auto fetch = [&](int i0, uint4(&y)[B][2]) {
#pragma unroll
                for (int i = 0; i < B && i0 + i < G; i++)
#pragma unroll
                    for (int k = 0; k < 2; k++) y[i][k] = load(from, 32 * tid + 16 * k, 32 * NT * (i0 + i));
            };
            fetch(0, raw[0]);
#pragma unroll
            for (int i0 = 0; i0 < G; i0 += B) {
                uint4(&y)[B][2] = raw[(i0 / B) & 1];
                __builtin_amdgcn_sched_barrier(0);
                if (i0 + B < G) fetch(i0 + B, raw[(i0 / B + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < B && i0 + i < G; i++) {
                    uint32_t high[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint4 q = y[i][e >> 1];
                        const uint64_t u = (e & 1 ? (uint64_t)q.w << 32 | q.z : (uint64_t)q.y << 32 | q.x) - ref;
                        x[4 * (i0 + i) + e] = (uint32_t)u;
                        high[e] = (uint32_t)(u >> 32);
                    }
                    if (edge(i0 + i)) {
#pragma unroll
                        for (int e = 0; e < 4; e++) high[e] = inside(symbol(i0 + i, e)) ? high[e] : 0;
                    }
                    apart |= (high[0] | high[1]) | (high[2] | high[3]);
                    take(i0 + i);
                }
            }
            if (__syncthreads_or(apart != 0)) {  // logits that lie further apart: uniform
                score_any_row<SRC, NW>(a, r, slots);
                return;
            }
        }
        const X m = block_join<NW>(mx, slots, Max());
        top_logit = SRC == SCORE_I32 ? (int64_t)m : (int64_t)((uint64_t)m + ref);
        if (some) {
            const uint64_t d = (uint64_t)top_logit - (uint64_t)of_token;
            td = d < (uint64_t)last ? (int)d : last;
        }
#pragma unroll
        for (int i = 0; i < 2 * G; i++) {
            uint32_t d[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t y = (uint32_t)m - (uint32_t)x[2 * i + e];  // (unsigned: any two)
                d[e] = y < cap ? y : cap;
            }
            d2[i] = d[0] | d[1] << 16;
        }
    }
    auto index = [&](int i, int e) { return e & 1 ? d2[2 * i + (e >> 1)] >> 16 : d2[2 * i + (e >> 1)] & 0xffffu; };
#pragma unroll
    for (int i = 0; i < G; i++)
        if (edge(i)) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = inside(symbol(i, e)) ? index(i, e) : cap;
            d2[2 * i] = y[0] | y[1] << 16;
            d2[2 * i + 1] = y[2] | y[3] << 16;
        }
    // (hides the pairs from the optimizer, which would keep every index unpacked from one walk to the next)
    auto hide = [&] {
#pragma unroll
        for (int i = 0; i < 2 * G; i++) asm volatile("" : "+v"(d2[i]));
    };
    hide();
#pragma unroll
    for (int i = 0; i < G; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) atomicAdd(&s_hist[index(i, e)], 1u);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    // fn(symbol, index) for the symbols with an index in lo ..= hi, few: a test a group of four
    auto those = [&](uint32_t lo, uint32_t hi, auto fn) {
        hide();
        const uint32_t span = (hi >= (uint32_t)last ? 0xffffu : hi) - lo;
#pragma unroll
        for (int i = 0; i < G; i++) {
            uint32_t p0 = d2[2 * i], p1 = d2[2 * i + 1], least = 0xffffffffu;
#pragma unroll
            for (int e = 0; e < 4; e++) least = index(i, e) - lo < least ? index(i, e) - lo : least;
            if (least > span) continue;
            asm volatile("" : "+v"(p0), "+v"(p1));  // (else the choice below makes an array in memory of all pairs)
#pragma unroll 1
            for (int e = 0; e < 4; e++) {
                const uint32_t d = ((e & 2 ? p1 : p0) >> (16 * (e & 1))) & 0xffffu;
                if (d - lo <= span && inside(symbol(i, e))) fn(symbol(i, e), d < (uint32_t)last ? (int)d : last);
            }
        }
    };
    __syncthreads();  // the counts are there
    if (w == 0) {     // the spare bins to the last one, without the places past the row
        const uint32_t far = (uint32_t)wave_sum64(s_hist[last + lane]);
        if (lane == 0) s_hist[last] = far - (uint32_t)(4 * G * NT - V);
    }
    uint32_t ahead = 0;  // symbols before the token
    __syncthreads();
    if (a.rank && some && s_hist[td] > 1) those((uint32_t)td, (uint32_t)td, [&](int j, int) { ahead += j < (int)token; });  // its ties
    // T and the entropy from the counts, in one pass: with w0 = table[0], the largest weight there is, the entropy
    // sum (w / T) ln(T / w) = ln(T / w0) + (sum w ln(w0 / w)) / T, two terms that are not negative (log_share takes the first,
    // exact where T is close to w0). In f32 the logarithms of the second are some 2^-22 off, which the first outweighs: it is
    // at least the share of all symbols but the largest.
    const uint64_t w0 = a.table[0];
    const float w0f = (float)w0;
    uint64_t sum = 0;
    float spread = 0;
    for (int d0 = tid; d0 <= last; d0 += 8 * NT) {
        uint32_t n[8];
        uint64_t x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int d = d0 + NT * k;
            n[k] = d <= last ? s_hist[d] : 0;
            x[k] = n[k] ? a.table[d] : 0;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            sum += n[k] * x[k];
            const float y = (float)x[k], l = __builtin_amdgcn_logf(w0f * __builtin_amdgcn_rcpf(y));
            spread += x[k] ? (float)n[k] * y * l : 0.0f;
            ahead += d0 + NT * k < td ? n[k] : 0;
        }
    }
    double h = (double)spread * 0.693147180559945309;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) h += __shfl_xor(h, o, 64);
    sum = wave_sum_dpp(sum);
    ahead = (uint32_t)wave_sum_dpp(ahead);
    if (lane == 0) s_sum[w] = sum, s_ahead[w] = ahead, s_ent[w] = h;
    const bool tops = a.top > 0 && (a.top_tokens || a.top_logprob);
    // the index up to which `top` symbols lie, and how many lie up to it: the last wave over 256 bins at a time
    if (tops && w == NW - 1) {
        uint32_t before = 0;
        for (int k0 = 0; k0 <= last; k0 += 256) {
            uint32_t c[4], mine = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                c[k] = k0 + 4 * lane + k <= last ? s_hist[k0 + 4 * lane + k] : 0;
                mine += c[k];
            }
            uint32_t upto = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(upto, o, 64);
                if (lane >= o) upto += y;
            }
            const uint64_t reached = __ballot(before + upto >= (uint32_t)a.top);
            if (reached) {  // (top <= vocab: some bin does)
                if (lane == __ffsll((unsigned long long)reached) - 1) {
                    uint32_t y = before + upto - mine;
                    int k = -1;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (y < (uint32_t)a.top) y += c[i], k = i;
                    s_thr = (uint32_t)(k0 + 4 * lane + k);
                    s_found = y;
                }
                break;
            }
            before += __shfl(upto, 63, 64);
        }
    }
    __syncthreads();
    uint64_t T = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) T += s_sum[i];
    if (tid == 0) {
        for (int i = 1; i < NW; i++) ahead += s_ahead[i], h += s_ent[i];
        if (a.logprob || a.rank) put_token(a, r, some, some ? a.table[td] : 0, T, ahead);
        if (a.entropy) a.entropy[r] = (float)(h / (double)T - log_share(w0, T));
    }
    if (!tops) return;
    const uint32_t thr = s_thr;
    if (s_found <= SCORE_LIST) {  // uniform
        those(0, thr, [&](int j, int d) { s_list[atomicAdd(&s_count, 1u)] = (uint64_t)d << 32 | (uint32_t)j; });
        __syncthreads();
        const int found = (int)s_found;
        for (int i = tid; i < found; i += NT) {
            const uint64_t x = s_list[i];
            int place = 0;
            for (int k = 0; k < found; k++) place += s_list[k] < x;
            if (place < a.top) put_top(a, r, place, (uint32_t)x, (int)(x >> 32), T);
        }
        return;
    }
    search_top<SRC, NW>(a, r, top_logit, T, slots);
}

template <int SRC, int G, int NW>
static hipError_t launch_score_rows(const ScoreArgs &a, int n_rows, hipStream_t stream) {
    const size_t lds = 4 * ((size_t)a.table_len + 63);
    const hipError_t e = allow_dynamic_lds((const void *)k_score_rows<SRC, G, NW>, lds);
    if (e != hipSuccess) return e;
    launch_k((k_score_rows<SRC, G, NW>), dim3(n_rows), dim3(64 * NW), lds, stream, a);
    return hipGetLastError();
}

template <int SRC>
static hipError_t launch_score_src(const ScoreArgs &a, int n_rows, hipStream_t stream) {
    if (a.table_len <= SCORE_BINS) {
        const int v = a.vocab + 3;  // with the part of 16 bytes before a row
        if (v <= 4 * 128 * 4) return launch_score_rows<SRC, 4, 2>(a, n_rows, stream);
        if (v <= 4 * 512 * 8) return launch_score_rows<SRC, 8, 8>(a, n_rows, stream);
        if constexpr (SRC == SCORE_I64) {
            if (v <= 4 * 1024 * 13) return launch_score_rows<SRC, 13, 16>(a, n_rows, stream);
        } else {
            if (v <= 4 * 512 * 26) return launch_score_rows<SRC, 26, 8>(a, n_rows, stream);
            if (v <= 4 * 1024 * 26) return launch_score_rows<SRC, 26, 16>(a, n_rows, stream);
        }
    }
    launch_k(k_score_any<SRC>, dim3(n_rows), dim3(512), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_score(const ScoreArgs &a, int n_rows, hipStream_t stream) {
    if (n_rows <= 0) return hipSuccess;
    if (a.src == SCORE_I32) return launch_score_src<SCORE_I32>(a, n_rows, stream);
    if (a.src == SCORE_I64) return launch_score_src<SCORE_I64>(a, n_rows, stream);
    return launch_score_src<SCORE_COMPACT>(a, n_rows, stream);
}

}  // namespace hs
