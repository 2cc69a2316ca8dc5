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
// and once for each alternative. The table's entries come from the L2, a symbol at a time: 64 rows of 50,257 symbols, 8 alternatives
// and 20,000 entries 272 us, where the histogram of shorter tables takes 18.6.
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

// A row by a workgroup of NW waves, its symbols four to a lane in groups of 256 NW. Each symbol's table index is counted in an
// LDS histogram; those past the table's end (and the places of the last group past the row) go to 64 spare bins, each lane's in
// its own, so that no symbol needs a test and none of these many collide. The counts give T, the entropy and the token's
// rank but for ties; one wave walks them for the index up to which the alternatives lie, and the symbols up to there, few, are
// collected and ranked against each other.
// G > 0: the row is read once, G groups at most, and its indexes stay in registers, 16 bits each. G > 26: the logits do not fit
// there until the largest is known, so 16 bits of each are kept (NARROW); a row whose largest logit lies too far above that
// of its first groups for those (65,535 less the table and 64) is scored by itself, as by k_score_any: slow (512 rows of 131,072
// whose first 16,384 symbols lie 100,000 below the others: 0.74 ms with one alternative and 6.8 with 64, others 99 and 109 us).
// G = 0, longer rows: read for the max, for the counts, and once each for ties and alternatives.
// HBM bounds many rows: 4,096 x 50,257 i32 logits, 823 MB in 182 us, 4.5 TB/s, with 53 us of LDS work (counting: over half of it
// waits for a bank) and 83 of VALU issue beside the loads of the other workgroup of a CU. Few rows are a chain: the loads, the
// largest, the counts, the sums, the alternatives: one row 17 us, 64 rows 17.7.
// Some forms spill registers: 13 groups of i64 logits 14, those of 16 bits each 25 (i32) and 30, the walk 24 and 42.
constexpr int SCORE_LIST = 1024;   // symbols collected; where ties make them more, the alternatives are searched one by one
constexpr int SCORE_BINS = 16384;  // entries of the table at most

template <int SRC, int G, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(4))) void k_score_rows(ScoreArgs a) {
    constexpr int NT = 64 * NW, LIST = NW == 1 ? 256 : SCORE_LIST;
    constexpr bool NARROW = SRC != SCORE_COMPACT && G > 26;  // the logits themselves do not fit the registers: 16 bits of each
    constexpr int GS = G && !NARROW ? G : 1;
    extern __shared__ uint32_t s_hist[];  // [table_len + 63]
    __shared__ uint64_t slots[NW], s_sum[NW], s_list[LIST], s_best[64];
    __shared__ double s_ent[NW];
    __shared__ uint32_t s_ahead[NW], s_count, s_thr, s_found, s_below;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.vocab, last = a.table_len - 1;
    const size_t r = blockIdx.x;
    const uint32_t cap = (uint32_t)(last + lane);  // this lane's bin of what lies past the table's end
    const ScoreRow<SRC> row(a, (int)r);

    // i32 logits as they are, i64 ones as their difference to 2^31 below the row's first one, in 32 bits; read 16 bytes at a
    // time, from the 16 bytes that the row starts in to those that it ends in (zeros past them). Compact ones in whole tiles.
    typedef typename std::conditional<SRC == SCORE_I64, uint32_t, int32_t>::type X;
    constexpr X LOW = SRC == SCORE_I64 ? (X)0 : (X)INT32_MIN;
    constexpr int E = SRC == SCORE_I64 ? 8 : SRC == SCORE_I32 ? 4 : 2;
    const uintptr_t at = SRC == SCORE_COMPACT ? (uintptr_t)(a.d16 + r * a.ld16) : (uintptr_t)a.logits + r * a.ld * E;
    const int off = SRC == SCORE_COMPACT ? 0 : (int)(at % 16) / E;  // symbol of element e of group i: 4 (NT i + tid) + e - off
    const auto from = __builtin_amdgcn_make_buffer_rsrc((void *)(at - at % 16), 0, SRC == SCORE_COMPACT ? (V + 63) / 64 * 128 : ((off + V) * E + 15) / 16 * 16, 0x00020000);
    const int groups = SRC == SCORE_COMPACT ? 2 * ((V + 8 * NT - 1) / (8 * NT)) : (V + off + 4 * NT - 1) / (4 * NT);
    // (compact ones eight together, two groups: they share a tile)
    auto symbol = [&](int i, int e) {
        return SRC == SCORE_COMPACT ? 8 * (NT * (i >> 1) + tid) + 4 * (i & 1) + e : 4 * (NT * i + tid) + e - off;
    };
    auto inside = [&](int j) { return j >= 0 && j < V; };
    auto edge = [&](int i) {  // some of group i are past the row (uniform)
        return SRC == SCORE_COMPACT ? 8 * NT * ((i >> 1) + 1) > V : (i == 0 && off > 0) || 4 * NT * (i + 1) > V + off;
    };
    typedef typename std::conditional<SRC == SCORE_I64, v4i[2], typename std::conditional<SRC == SCORE_I32, v4i[1], v2i[1]>::type>::type Raw;
    // Groups past the row are loaded too (zeros without an access): the place in the lane's offset, which the descriptor's end
    // bounds. A scalar offset is not part of that check.
    int place = SRC == SCORE_COMPACT ? 16 * tid : 4 * E * tid;
    if constexpr (SRC == SCORE_COMPACT) asm volatile("" : "+v"(place));  // (hidden from the optimizer: it would keep all groups' places)
    auto fetch = [&](int i, Raw &y) {
        if constexpr (SRC == SCORE_COMPACT) {
            y[0] = __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(from, place + 16 * NT * (i >> 1) + 8 * (i & 1), 0, 0));
        } else {
#pragma unroll
            for (int k = 0; k < E / 4; k++)
                y[k] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(from, place + 4 * E * NT * i + 16 * k, 0, 0));
        }
    };
    uint64_t ref = 0;
    uint32_t apart = 0;  // not 0: the differences do not fit
    auto start = [&] {   // (behind the first loads)
        if constexpr (SRC == SCORE_I64) {
            const int64_t first = *(const int64_t *)at;
            if (first >= (int64_t)1 << 62 || first < -((int64_t)1 << 62)) apart = 1;  // (they would come round)
            ref = (uint64_t)first - 0x80000000u;
        }
        for (int k = tid; k < last + 64; k += NT) s_hist[k] = 0;
        if (tid == 0) s_count = 0;
    };
    X mx = LOW;
    auto values = [&](int i, const Raw &y, X (&x)[4]) {
        if constexpr (SRC == SCORE_I64) {
            uint32_t high[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint64_t u = ((uint64_t)(uint32_t)y[e >> 1][2 * (e & 1) + 1] << 32 | (uint32_t)y[e >> 1][2 * (e & 1)]) - ref;
                x[e] = (X)u;
                high[e] = (uint32_t)(u >> 32);
            }
            if (edge(i)) {
#pragma unroll
                for (int e = 0; e < 4; e++) high[e] = inside(symbol(i, e)) ? high[e] : 0;
            }
            apart |= (high[0] | high[1]) | (high[2] | high[3]);
        } else if constexpr (SRC == SCORE_I32) {
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = y[0][e];
        }
        if (edge(i)) {
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = inside(symbol(i, e)) ? x[e] : LOW;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) mx = x[e] > mx ? x[e] : mx;
    };

    X x[GS][4];
    X base = LOW;
    uint32_t d2[2 * (G ? G : 1)];  // G > 0: the indexes, pairs
    Raw raw[SRC == SCORE_COMPACT ? GS : 1];
    int64_t tile[SRC == SCORE_COMPACT ? GS : 1];
    const int64_t *tm = a.tmax + r * a.ntiles;
    auto tile_of = [&](int i) { return tm[symbol(i, 0) < V ? symbol(i, 0) >> 6 : 0]; };
    if constexpr (SRC == SCORE_COMPACT) {
        if constexpr (G > 0) {
#pragma unroll
            for (int i = 0; i < G; i++) {
                fetch(i, raw[i]);
                tile[i] = i & 1 ? tile[i - 1] : tile_of(i);
            }
        }
        start();
    } else if constexpr (NARROW) {
        // The largest logit is not known yet, but no smaller than that of the first groups, M0: what lies last + 64 below M0 or
        // more is past the table, and the others are kept as their difference to that, where 16 bits hold it.
        constexpr int B = SRC == SCORE_I32 ? 4 : 2;  // groups in flight, besides those at work
        Raw y[2][B];
#pragma unroll
        for (int i = 0; i < B; i++) fetch(i, y[0][i]);
        __builtin_amdgcn_sched_barrier(0);
        start();
        auto keep = [&](int i, const X (&v)[4]) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = (uint32_t)(v[e] > base ? v[e] : base) - (uint32_t)base;
            apart |= ((u[0] | u[1]) | (u[2] | u[3])) >> 16;
            d2[2 * i] = (u[0] & 0xffffu) | u[1] << 16;
            d2[2 * i + 1] = (u[2] & 0xffffu) | u[3] << 16;
            // (hidden from the optimizer: it would put this off and keep the logits)
            asm volatile("" : "+v"(d2[2 * i]), "+v"(d2[2 * i + 1]), "+v"(apart), "+v"(mx));
        };
#pragma unroll
        for (int i0 = 0; i0 < G; i0 += B) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = i0 + B; i < i0 + 2 * B && i < G; i++) fetch(i, y[(i0 / B + 1) & 1][i - i0 - B]);
            __builtin_amdgcn_sched_barrier(0);
            X v[B][4];
#pragma unroll
            for (int i = i0; i < i0 + B && i < G; i++) values(i, y[(i0 / B) & 1][i - i0], v[i - i0]);
            if (i0 == 0) {
                const X M0 = block_join<NW>(mx, slots, Max());
                base = M0 > (X)(LOW + last + 64) ? (X)(M0 - last - 64) : LOW;
            }
#pragma unroll
            for (int i = i0; i < i0 + B && i < G; i++) keep(i, v[i - i0]);
        }
    } else if constexpr (G > 0) {
        constexpr int B = SRC == SCORE_I32 ? G : 4;  // groups in flight, besides those at work (i32: all)
        Raw y[2][B];
#pragma unroll
        for (int i = 0; i < B && i < G; i++) fetch(i, y[0][i]);
        __builtin_amdgcn_sched_barrier(0);
        start();
#pragma unroll
        for (int i0 = 0; i0 < G; i0 += B) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = i0 + B; i < i0 + 2 * B && i < G; i++) fetch(i, y[(i0 / B + 1) & 1][i - i0 - B]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = i0; i < i0 + B && i < G; i++) values(i, y[(i0 / B) & 1][i - i0], x[i]);
        }
    } else {
        start();
        for (int i0 = 0; i0 < groups; i0 += 8) {
            Raw y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) fetch(i0 + i, y[i]);
#pragma unroll
            for (int i = 0; i < 8; i++) values(i0 + i, y[i], x[0]);
        }
    }
    const uint64_t w0 = a.table[0];
    const uint32_t token = a.tokens ? a.tokens[r] : 0xffffffffu;
    const bool some = token < (uint32_t)V;
    const int64_t of_token = SRC != SCORE_COMPACT && some ? row.value((int)token) : 0;
    int64_t M;
    if constexpr (SRC == SCORE_COMPACT) {
        int64_t most = INT64_MIN;
        for (int j = tid; j < a.ntiles; j += NT) most = tm[j] > most ? tm[j] : most;
        M = block_join<NW>(most, slots, Max());
    } else {
        mx = block_join<NW>(mx, slots, Max());  // (its barriers: the histogram is clear)
        M = SRC == SCORE_I32 ? (int64_t)mx : (int64_t)((uint64_t)(uint32_t)mx + ref);
    }
    // logits that lie further apart; and a table that is not a model's (the entropy below divides by w0): uniform
    if (w0 == 0 || ((SRC == SCORE_I64 || NARROW) && __syncthreads_or(apart != 0))) {
        score_any_row<SRC, NW>(a, r, slots);
        return;
    }
    int td = 0;  // the token's index
    if (some) {
        if constexpr (SRC == SCORE_COMPACT) {
            td = row.index(M, (int)token);
        } else {
            const uint64_t d = (uint64_t)M - (uint64_t)of_token;
            td = d < (uint64_t)last ? (int)d : last;
        }
    }
    // the indexes of a group, cap for what lies past the table and the row
    auto indexes = [&](int i, const Raw &y, const X (&v)[4], int64_t t, uint32_t (&d)[4]) {
        if constexpr (SRC == SCORE_COMPACT) {
            const uint64_t b = (uint64_t)M - (uint64_t)t;
            const unsigned short base = (unsigned short)(b < (uint64_t)cap ? (uint32_t)b : cap);
#pragma unroll
            for (int k = 0; k < 2; k++) {  // (a d16 may be capped at last: past the table too)
                const int two = y[0][k];
                us2 p;
                __builtin_memcpy(&p, &two, 4);
                p = __builtin_elementwise_min(__builtin_elementwise_add_sat(p, us2{base, base}), us2{(unsigned short)cap, (unsigned short)cap});
                d[2 * k] = p.x;
                d[2 * k + 1] = p.y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                d[e] = (uint32_t)mx - (uint32_t)v[e];  // (unsigned: any two)
                d[e] = d[e] < cap ? d[e] : cap;
            }
        }
        if (edge(i)) {
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = inside(symbol(i, e)) ? d[e] : cap;
        }
    };
    uint32_t places = 0;  // counted
    if constexpr (NARROW) {
        const uint32_t most = (uint32_t)mx - (uint32_t)base;
#pragma unroll
        for (int i = 0; i < G; i++) {
            uint32_t d[4] = {cap, cap, cap, cap};
            if (i < groups) {  // uniform
                const uint32_t q[2] = {d2[2 * i], d2[2 * i + 1]};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t u = most - (e & 1 ? q[e >> 1] >> 16 : q[e >> 1] & 0xffffu);
                    d[e] = u < cap ? u : cap;
                }
                if (edge(i)) {
#pragma unroll
                    for (int e = 0; e < 4; e++) d[e] = inside(symbol(i, e)) ? d[e] : cap;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) atomicAdd(&s_hist[d[e]], 1u);
            }
            d2[2 * i] = d[0] | d[1] << 16;
            d2[2 * i + 1] = d[2] | d[3] << 16;
            __builtin_amdgcn_sched_barrier(0);
        }
        places = 4 * NT * groups;
    } else if constexpr (G > 0) {
#pragma unroll
        for (int i = 0; i < G; i++) {
            uint32_t d[4];
            indexes(i, raw[SRC == SCORE_COMPACT ? i : 0], x[i], tile[SRC == SCORE_COMPACT ? i : 0], d);
#pragma unroll
            for (int e = 0; e < 4; e++) atomicAdd(&s_hist[d[e]], 1u);
            d2[2 * i] = d[0] | d[1] << 16;
            d2[2 * i + 1] = d[2] | d[3] << 16;
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        places = 4 * G * NT;
    }
    // fn(i, y): the loads of each group (G = 0), eight at a time, and its values and tile maxes
    auto walk = [&](auto fn) {
        for (int i0 = 0; i0 < groups; i0 += 8) {
            Raw y[8];
            int64_t t[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                fetch(i0 + i, y[i]);
                if constexpr (SRC == SCORE_COMPACT) t[i] = i & 1 ? t[i - 1] : tile_of(i0 + i);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                uint32_t d[4];
                X v[4];
                if (i0 + i >= groups) break;  // uniform
                if constexpr (SRC != SCORE_COMPACT) values(i0 + i, y[i], v);
                indexes(i0 + i, y[i], v, t[i], d);
                fn(i0 + i, d);
            }
        }
    };
    if constexpr (G == 0) {
        walk([&](int, uint32_t (&d)[4]) {
#pragma unroll
            for (int e = 0; e < 4; e++) atomicAdd(&s_hist[d[e]], 1u);
        });
        places = 4 * NT * groups;
    }
    // fn(symbol, index) for the symbols with an index in lo ..= hi, few: a test for eight at once
    auto those = [&](uint32_t lo, uint32_t hi, auto fn) {
        const uint32_t span = (hi >= (uint32_t)last ? 0xffffu : hi) - lo;
        auto take = [&](int i, int e, uint32_t d) {
            if (d - lo <= span && inside(symbol(i, e))) fn(symbol(i, e), d < (uint32_t)last ? (int)d : last);
        };
        if constexpr (G == 0) {
            walk([&](int i, uint32_t (&d)[4]) {
#pragma unroll
                for (int e = 0; e < 4; e++) take(i, e, d[e]);
            });
        } else {
            const us2 base = {(unsigned short)lo, (unsigned short)lo}, most = {(unsigned short)span, (unsigned short)span};
#pragma unroll
            for (int i = 0; i < G; i += 2) {
                uint32_t q[4];
                us2 least = {0xffff, 0xffff};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    q[k] = 2 * i + k < 2 * G ? d2[2 * i + k] : 0xffffffffu;
                    // (hidden from the optimizer: it would keep the indexes unpacked from one walk to the next, or make an array
                    // in memory for the choice below)
                    asm volatile("" : "+v"(q[k]));
                    us2 p;
                    __builtin_memcpy(&p, &q[k], 4);
                    p -= base;
                    least = __builtin_elementwise_min(least, p);
                }
                const us2 over = __builtin_elementwise_sub_sat(least, most);  // 0: one of the four lies in the span
                if (over.x && over.y) continue;
#pragma unroll 1
                for (int e = 0; e < 8; e++) {
                    const uint32_t pair = e & 4 ? (e & 2 ? q[3] : q[2]) : (e & 2 ? q[1] : q[0]);
                    take(i + (e >> 2), e & 3, (pair >> (16 * (e & 1))) & 0xffffu);
                }
            }
        }
    };
    __syncthreads();  // the counts are there
    if (w == 0) {     // the spare bins to the last one, without the places past the row
        const uint32_t far = (uint32_t)wave_sum_dpp(s_hist[last + lane]);
        if (lane == 0) s_hist[last] = far - (places - (uint32_t)V);
    }
    uint32_t ahead = 0;  // symbols before the token
    __syncthreads();
    if (a.rank && some && s_hist[td] > 1) {  // its ties (uniform)
        if (G > 0 && s_hist[td] > 512) {     // many, those past the table say: without a branch
            const uint32_t span = (td >= last ? 0xffffu : (uint32_t)td) - (uint32_t)td;
#pragma unroll
            for (int i = 0; i < G; i++) {
                uint32_t q[2] = {d2[2 * i], d2[2 * i + 1]};
                asm volatile("" : "+v"(q[0]), "+v"(q[1]));
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t d = e & 1 ? q[e >> 1] >> 16 : q[e >> 1] & 0xffffu;
                    ahead += d - (uint32_t)td <= span && (uint32_t)symbol(i, e) < token;
                }
            }
        } else {
            those((uint32_t)td, (uint32_t)td, [&](int j, int) { ahead += j < (int)token; });
        }
    }
    // T and the entropy from the counts, in one pass: with w0 = table[0], the largest weight there is, the entropy
    // sum (w / T) ln(T / w) = ln(T / w0) + (sum w ln(w0 / w)) / T, two terms that are not negative (log_share takes the first,
    // exact where T is close to w0). Symbols of weight w0 add exactly nothing to the second. For each of the others the quotient
    // and its logarithm in f32 are at most 3.5 2^-23 + 2^-23 ln(w0 / w) off, the product with the weight 2^-22 of itself, and
    // the sum is in f64: some 2^-21 of the entropy in all, since the first term is at least the share of those others.
    const float w0f = (float)w0;
    uint64_t sum = 0;
    double spread = 0;
    for (int d0 = tid; d0 <= last; d0 += 8 * NT) {
        uint32_t n[8];
        uint64_t z[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int d = d0 + NT * k;
            n[k] = d <= last ? s_hist[d] : 0;
            z[k] = n[k] ? a.table[d] : 0;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            sum += n[k] * z[k];
            const float y = fmaf((float)(uint32_t)(z[k] >> 32), 0x1p32f, (float)(uint32_t)z[k]);
            const float l = __builtin_amdgcn_logf(w0f * __builtin_amdgcn_rcpf(y));
            spread += (double)(z[k] && z[k] != w0 ? (float)n[k] * y * l : 0.0f);
            ahead += d0 + NT * k < td ? n[k] : 0;
        }
    }
    double h = spread * 0.693147180559945309;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) h += __shfl_xor(h, o, 64);
    sum = wave_sum_dpp(sum);
    ahead = (uint32_t)wave_sum_dpp(ahead);
    if (lane == 0) s_sum[w] = sum, s_ahead[w] = ahead, s_ent[w] = h;
    const bool tops = a.top > 0 && (a.top_tokens || a.top_logprob);
    // the index up to which `top` symbols lie, and how many lie up to it: the last wave over 1,024 bins at a time
    if (tops && w == NW - 1) {
        uint32_t before = 0;
        for (int k0 = 0; k0 <= last; k0 += 1024) {
            uint32_t c[16], mine = 0;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                c[k] = k0 + 16 * lane + k <= last ? s_hist[k0 + 16 * lane + k] : 0;
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
                    uint32_t y = before + upto - mine, under = 0;
                    int k = -1;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (y < (uint32_t)a.top) under = y, y += c[i], k = i;
                    s_thr = (uint32_t)(k0 + 16 * lane + k);
                    s_found = y;
                    s_below = under;
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
    int best = 0;  // alternatives in s_best
    if (tops) {
        const uint32_t thr = s_thr;
        const bool ties = s_found > LIST;  // more than the list holds, so most of them equal: those of thr apart (uniform)
        if (!ties || thr > 0)
            those(0, ties ? thr - 1 : thr, [&](int j, int d) { s_list[atomicAdd(&s_count, 1u)] = (uint64_t)d << 32 | (uint32_t)j; });
        __syncthreads();
        const int found = (int)(ties ? s_below : s_found);
        for (int i = tid; i < found; i += NT) {
            const uint64_t one = s_list[i];
            int place = 0;
            for (int k = 0; k < found; k++) place += s_list[k] < one;
            if (place < a.top) s_best[place] = one;
        }
        if (ties) {  // the first of the equal ones, in the symbols' order
            for (int j0 = 0, got = found; got < a.top && j0 < V; j0 += NT) {
                const bool in = j0 + tid < V && row.index(M, j0 + tid < V ? j0 + tid : 0) == (int)thr;
                const uint64_t m = __ballot(in);
                if (lane == 0) slots[w] = (uint64_t)__popcll(m);
                __syncthreads();
                int place = got + __popcll(m & (((uint64_t)1 << lane) - 1));
#pragma unroll
                for (int i = 0; i < NW; i++) {
                    place += i < w ? (int)slots[i] : 0;
                    got += (int)slots[i];
                }
                if (in && place < a.top) s_best[place] = (uint64_t)thr << 32 | (uint32_t)(j0 + tid);
                __syncthreads();
            }
        }
        __syncthreads();
        best = a.top;
    }
    // one logarithm a lane: the alternatives', the token's, the entropy's
    for (int i = tid; i < best + 2; i += NT) {
        const uint64_t one = i < best ? s_best[i] : 0;
        const uint64_t weight = i < best ? a.table[one >> 32] : i == best ? (some ? a.table[td] : 1) : w0;
        const double l = log_share(weight, T);
        if (i < best) {
            if (a.top_tokens) a.top_tokens[r * a.top + i] = (uint32_t)one;
            if (a.top_logprob) a.top_logprob[r * a.top + i] = (float)l;
        } else if (i == best) {
            uint32_t n = 0;
            for (int k = 0; k < NW; k++) n += s_ahead[k];
            if (a.logprob) a.logprob[r] = some ? (float)l : 0.0f;
            if (a.rank) a.rank[r] = some ? n : 0xffffffffu;
        } else if (a.entropy) {
            double x = 0;
            for (int k = 0; k < NW; k++) x += s_ent[k];
            a.entropy[r] = (float)(x / (double)T - l);
        }
    }
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
        // As many waves as the row has groups for, in us: 3,001 rows of 299 symbols by one wave 13.6, by eight 63; 512 rows of
        // 16,000 by eight 19.8, by sixteen 31.8. Rows of 50,257: more rows than CUs share them, one workgroup at its loads while
        // another counts (4,096 rows: 26 groups of eight waves 181, 13 of sixteen 251; 512 rows 35.9 and 42.4), fewer take a CU
        // each (64 rows 18.6 and 21); i64 groups are twice the loads, and 26 of them do not fit the registers. The walk takes 451
        // for the 4,096 rows, and 120 for 512 of i64 (74). Longer rows in 16 bits each, and walked: 512 of 131,072 103 and 163,
        // 1,024 of 60,000 i64 183 and 264, one of 131,072 27 and 34.
        const int v = a.vocab + 3;  // with the part of 16 bytes before a row
        if (v <= 4 * 64 * 4) return launch_score_rows<SRC, 4, 1>(a, n_rows, stream);
        if (v <= 4 * 512 * 8) return launch_score_rows<SRC, 8, 8>(a, n_rows, stream);
        if constexpr (SRC == SCORE_I64) {
            if (v <= 4 * 1024 * 13) return launch_score_rows<SRC, 13, 16>(a, n_rows, stream);
        } else {
            if (n_rows <= 256 && v <= 4 * 1024 * 13) return launch_score_rows<SRC, SRC == SCORE_COMPACT ? 14 : 13, 16>(a, n_rows, stream);
            if (v <= 4 * 512 * 26) return launch_score_rows<SRC, 26, 8>(a, n_rows, stream);
        }
        if constexpr (SRC != SCORE_COMPACT)
            if (v <= 4 * 1024 * 33) return launch_score_rows<SRC, 33, 16>(a, n_rows, stream);
        return launch_score_rows<SRC, 0, 16>(a, n_rows, stream);
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
