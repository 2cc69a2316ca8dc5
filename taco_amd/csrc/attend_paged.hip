// Attention over pages of 8-bit keys and values with a scale for each page and head (no counterpart in the
// reference): score_j = clamp(rescale(q k_j, score_m ks, score_s), +-2^40), e_j = table[min(M - score_j, len - 1)],
// S = sum e_j, w_j = floor(e_j vs 2^P / S), out = clamp(rescale(sum w_j v_j, out_m, out_s), +-127), with ks and vs the
// scales of key j's page: the rule of the other attention kernels where the scales are 1.
#include "attend.h"

namespace hs {

constexpr int PG_TABLE = 16384;  // entries of the table copied to LDS at most
constexpr int PG_ACC = 66;       // 64 channels' sums of a row and two of padding (bank spread)
constexpr int PG_NONE = 0x7fffffff;  // a lane's offset past any page: the buffer load gives zeros

struct PagedPlan {
    int rt = 16;               // rows of a tile
    int group = 1, tiles = 1;  // query heads of a cache head; row tiles of a panel
    int panels = 0;            // (stream, cache head)
    int ng = 1, span = 0;      // key ranges, their keys
    int store = 0;             // the ranges' scores are kept in the scratch
    int rows = 0, chunks = 1;  // rows of a tile with scores there; of PG_CHUNK keys, with a sum each
    int page_log = 4;
};
constexpr int PG_CHUNK = 4096;

// What the ranges leave for the next launch, for each tile of each panel.
struct PagedScratch {
    int64_t *mx;    // [ng][rt]: the largest score
    uint64_t *sum;  // [chunks or ng][rt]: the sum of the entries
    int64_t *part;  // [ng][rt][hd]: sum w v
    int64_t *keep;  // [rows][ng span]: the scores, then the entries, as i32 in half of it where they fit
};
__host__ __device__ inline size_t pg256(size_t x) { return (x + 255) / 256 * 256; }
__host__ __device__ inline PagedScratch paged_scratch(void *base, const PagedPlan &p, int hd, size_t *bytes = nullptr) {
    const size_t n = (size_t)p.panels * p.tiles;
    PagedScratch s;
    size_t at = 0;
    s.mx = (int64_t *)base;
    at += pg256(n * p.ng * p.rt * 8);
    s.sum = (uint64_t *)((char *)base + at);
    at += pg256(n * p.chunks * p.rt * 8);
    s.part = (int64_t *)((char *)base + at);
    at += pg256(n * p.ng * p.rt * hd * 8);
    s.keep = (int64_t *)((char *)base + at);
    if (p.store) at += pg256(n * p.rows * p.ng * p.span * 8);
    if (bytes) *bytes = at;
    return s;
}

// The score of a dot under a page's multiplier m = score_m ks (0 < m < 2^31), and the table index of another under the
// row's largest score M. HI (shifts of 32 to 60): |dot m| < 2^53, so the score is the high word of dot m + 2^(s-1) shifted
// by s - 32, an i32, and M - score that of -dot m + c, with one constant c a row (the rule of RowIndex).
template <bool HI>
struct PagedRule {
    int64_t half;
    int s;
    __device__ __forceinline__ explicit PagedRule(const PagedArgs &g)
        : half(g.score_s == 0 || g.score_s > 62 ? 0 : (int64_t)1 << (g.score_s - 1)), s(g.score_s < 63 ? g.score_s : 63) {}
    __device__ __forceinline__ int64_t score(int32_t dot, int32_t m) const {
        const int64_t x = (int64_t)dot * m + half;
        if constexpr (HI) return (int32_t)(x >> 32) >> (s - 32);
        else return clamp64(x >> s, -SCORE_LIMIT, SCORE_LIMIT);
    }
    __device__ __forceinline__ int64_t constant(int64_t M) const {
        if constexpr (HI) return (((M + 1) << (s - 32)) - 1) * ((int64_t)1 << 32) + 0xffffffffll - half;
        else return M;
    }
    __device__ __forceinline__ uint32_t index(int32_t dot, int32_t m, int64_t c, uint32_t last) const {
        if constexpr (HI) {
            const uint32_t i = (uint32_t)((int32_t)(((int64_t)dot * -m + c) >> 32) >> (s - 32));
            return i < last ? i : last;
        } else {
            return (uint32_t)clamp64(c - score(dot, m), 0, last);
        }
    }
};

// Tiles of RT rows (16, or 4 where there are no more) of one (stream, cache head): row r is query head r % group of
// token r / group. Wave w takes the blocks of 64 keys w, w + NW, .. of the range, NB at most, each in four groups of 16
// keys that lie in one page. K is the first operand of v_mfma_i32_16x16x64_i8, so lane l holds dots of column l % 16
// with keys 4 (l / 16) + e of a group. With 16 rows a column is a row and D[t] holds group t. With 4 rows column 4 t + r is
// row r with group t: the products of the four groups add up in one accumulator, each with q in its own columns and
// zeros in the others, so that no lane idles; the product with V takes the rows' four digit planes as its 16 columns.
// PHASE 0: all in one launch. Else the ranges meet in the scratch: 1 the largest scores, 2 the sums of the entries, 3 the
// products with V. KEEP: launch 1 leaves all scores there (0x80.. where a row does not see a key), k_paged_entries makes them
// entries and sums, and launch 3 reads those; else each launch forms the dots again.
template <int RT, int QC, int NB, int NW, bool HI, int PHASE, bool KEEP>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW > 8 ? 4 : 2))) void k_paged_tile(PagedArgs g, PagedPlan pl, void *scratch) {
    static_assert(NB <= 16, "a lane for each group of the wave's blocks");
    static_assert(RT == 4 || NB <= 4, "two planes' sums of a wave's keys in 32 bits");
    constexpr int TU = RT / 4;  // accumulators of a block
    constexpr int KD = QC == 1 ? (NB < 4 ? NB : NW > 8 ? 2 : 4) : QC == 2 && NB > 1 && NW <= 8 ? 2 : 1;  // blocks of K in flight, and of V
    constexpr bool DOTS = !(KEEP && PHASE == 3);  // whether the launch forms the dots
    typedef typename std::conditional<HI, int32_t, int64_t>::type Score;
    constexpr Score LOW = HI ? (Score)INT32_MIN : (Score)INT64_MIN;
    extern __shared__ __attribute__((aligned(1024))) int8_t s_mem[];
    const PagePool &p = g.pages;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4, hd = p.hd;
    // workgroup L runs on XCD L % 8: the tiles of a panel stay on one XCD and share K and V in its L2
    const int inner = pl.tiles * pl.ng;
    const int L = blockIdx.x, panel = L / (8 * inner) * 8 + (L & 7), in = (L >> 3) % inner;
    if (panel >= pl.panels) return;
    const int tile = in % pl.tiles, range = in / pl.tiles;
    const int s = panel / p.kv_heads, h = panel - s * p.kv_heads;
    const int n = (int)(g.ctx[s] < (uint32_t)g.keys ? g.ctx[s] : (uint32_t)g.keys);  // the stream's keys
    uint32_t count = g.rows ? g.rows[s] : (uint32_t)g.t;
    count = count < (uint32_t)g.t ? count : (uint32_t)g.t;
    const int rows = (int)count * pl.group, row0 = RT * tile;
    if (row0 >= rows) return;
    const int live = rows - row0 < RT ? rows - row0 : RT;
    const int before = n - (int)count;  // token i sees keys up to before + i
    const int whole = before + row0 / pl.group + 1, keys = before + (row0 + live - 1) / pl.group + 1;
    const int k0 = PHASE ? range * pl.span : 0;
    if (PHASE && k0 >= keys && range > 0) return;  // the launches behind read no result of this range
    const int k1 = PHASE && k0 + pl.span < keys ? k0 + pl.span : keys;
    const int ranges = PHASE && keys > pl.span ? (keys + pl.span - 1) / pl.span : 1;
    const uint32_t last = (uint32_t)g.exp_len - 1;

    // LDS: the table (of 16 rows), which the sums of the outputs take over, each wave's V, what the waves exchange
    const bool in_lds = RT == 16 && PHASE != 1 && !(KEEP && PHASE == 3) && g.table_lds;
    constexpr int ACC_BYTES = (8 * QC * RT * PG_ACC + 1023) / 1024 * 1024;
    const int table_bytes = in_lds ? 1024 * ((g.exp_len + 255) / 256) : 0;
    const int top = table_bytes > ACC_BYTES ? table_bytes : ACC_BYTES;
    int32_t *s_exp = (int32_t *)s_mem;
    int64_t *s_acc = (int64_t *)s_mem;  // [QC][RT][PG_ACC]
    int8_t *s_v = s_mem + top + 4096 * w;
    uint64_t *s_sum = (uint64_t *)(s_mem + top + 4096 * NW);  // [NW][RT]
    int64_t *s_mx = (int64_t *)(s_sum + NW * RT);             // [NW][RT]
    if (in_lds) {
        for (int ch = w; ch < g.exp_len / 256; ch += NW)
            __builtin_amdgcn_global_load_lds((const void *)(g.exp_table + ch * 256 + 4 * lane), (lds_void *)(s_exp + ch * 256), 16, 0, 0);
        if (w == 0)
            for (int i = g.exp_len / 256 * 256 + lane; i < table_bytes / 4; i += 64) s_exp[i] = g.exp_table[i < g.exp_len ? i : g.exp_len - 1];
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);  // the table's loads before those of K: who has K has the table
    }

    // lane 4 j + t: the page of group t of the wave's block j, and its scales
    auto key_of = [&](int j) { return k0 + 64 * (NW * j + w); };
    auto mine = [&](int j) { return key_of(j) < k1; };  // uniform
    uint32_t number = 0xffffffffu, mul = 0, vs = 1;
    {
        const int key = key_of(lane >> 2) + 16 * (lane & 3);
        if ((lane >> 2) < NB && key < k1) number = g.table[(size_t)s * g.width + (key >> pl.page_log)];
    }
    const bool held = number < (uint32_t)p.pages;
    const uint64_t there = __ballot(held);  // of the groups, those with keys and a page
    if (held) {
        const size_t at = (size_t)number * p.kv_heads + h;
        if (DOTS) mul = p.k_scale[at];
        if (PHASE == 0 || PHASE == 3) vs = p.v_scale[at];
    }
    auto group_rows = [&](const int8_t *pool, int j, int t) {  // the 16 rows of a group; no access where they are not there
        const bool in_page = (there >> (4 * j + t)) & 1;
        const uint32_t page = in_page ? (uint32_t)__builtin_amdgcn_readlane((int)number, 4 * j + t) : 0;
        const size_t row = (((size_t)page * p.kv_heads + h) << pl.page_log) + ((key_of(j) + 16 * t) & (p.page - 1));
        return __builtin_amdgcn_make_buffer_rsrc((void *)(pool + row * hd), 0, in_page ? 16 * hd : 0, 0x00020000);
    };
    auto load = [&](__amdgpu_buffer_rsrc_t r, int at) { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0)); };
    // K as the product's operand (chunk c: bytes 64 c + 16 (l / 16) .. of row l % 16), V as block_pv's (16-byte chunk
    // l % 4, swizzled, of row l / 4); channels past the head are zeros
    auto k_load = [&](int j, v4i (&x)[4][QC]) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const auto r = group_rows(p.k, j, t);
#pragma unroll
            for (int c = 0; c < QC; c++) {
                const int o = 64 * c + 16 * qg;
                x[t][c] = load(r, o < hd ? ql * hd + o : PG_NONE);
            }
        }
    };
    auto v_load = [&](int j, int c, v4i (&x)[4]) {
        const int r = lane >> 2, o = 64 * c + 16 * ((lane & 3) ^ vsw<4>(r)), at = o < hd ? r * hd + o : PG_NONE;
#pragma unroll
        for (int t = 0; t < 4; t++) x[t] = load(group_rows(p.v, j, t), at);
    };

    const v4i zero = v4i{0, 0, 0, 0};
    const int row = RT == 16 ? ql : ql & 3, near = row < live ? row : live - 1;  // rows that are not there: as the last one
    const int64_t first = (int64_t)s * g.t;                                      // the stream's first token
    const size_t place = (size_t)panel * pl.tiles + tile, slot = place * pl.ng;   // of the tile, of its ranges
    const PagedScratch S = paged_scratch(scratch, pl, hd);
    // a lane's scores or entries of block j, accumulator u in the scratch: four keys of its row
    auto kept = [&](int j, int u) {
        const int key = key_of(j) + 16 * (RT == 16 ? u : ql >> 2) + 4 * qg;
        return (Score *)S.keep + (place * pl.rows + row) * ((size_t)pl.ng * pl.span) + key;
    };
    v4i D[NB][TU];
    v4i vr[KD][4];
    if constexpr (DOTS) {
        v4i qf[RT == 16 ? 1 : 4][QC];
        const int tok = (row0 + row) / pl.group, head = h * pl.group + (row0 + row) % pl.group;
#pragma unroll
        for (int c = 0; c < QC; c++) {
            const int o = 64 * c + 16 * qg;
            const v4i x = row < live && o < hd ? *(const v4i *)(g.q + (first + tok) * g.q_stride + (size_t)head * hd + o) : zero;
            if constexpr (RT == 16) {
                qf[0][c] = x;
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++) qf[t][c] = (ql >> 2) == t ? x : zero;
            }
        }
        // all loads without a branch around them, so that the waits count them exactly
        v4i kr[KD][4][QC];
#pragma unroll
        for (int j = 0; j < KD; j++) k_load(j, kr[j]);
        if constexpr (PHASE == 0 && NB <= KD) {
#pragma unroll
            for (int j = 0; j < NB; j++) v_load(j, 0, vr[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NB; j++) {
            v4i(&x)[4][QC] = kr[j % KD];
            if (mine(j)) {
#pragma unroll
                for (int u = 0; u < TU; u++) D[j][u] = zero;
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int c = 0; c < QC; c++) {
                        v4i &d = D[j][RT == 16 ? t : 0];
                        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[t][c], qf[RT == 16 ? 0 : t][c], d, 0, 0, 0);
                    }
            }
            if (j + KD < NB) k_load(j + KD, x);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int u = 0; u < TU; u++) {
                D[j][u] = zero;
                if (!mine(j) || row >= live) continue;
                if constexpr (HI) {
                    D[j][u] = *(const v4i *)kept(j, u);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) D[j][u][e] = (int32_t)kept(j, u)[e];
                }
            }
    }
    if constexpr ((PHASE == 0 && NB > KD) || PHASE == 3) {
#pragma unroll
        for (int j = 0; j < KD; j++) v_load(j, 0, vr[j]);
    }

    // which of a lane's keys its row sees, where not all do
    mul = (mul < 1 ? 1 : (mul > p.max_scale ? p.max_scale : mul)) * (uint32_t)g.score_m;
    vs = vs < 1 ? 1 : (vs > p.max_scale ? p.max_scale : vs);
    const int most = whole < k1 ? whole : k1;
    auto all = [&](int j) { return key_of(j) + 64 <= most && ((there >> (4 * j)) & 15) == 15; };  // uniform
    const int sees = before + (row0 + near) / pl.group + 1, lim = sees < k1 ? sees : k1;
    auto group_of = [&](int u) { return RT == 16 ? u : ql >> 2; };
    auto seen = [&](int j, int u) {  // how many of the lane's four keys
        const int x = lim - (key_of(j) + 16 * group_of(u) + 4 * qg);
        return (there >> (4 * j + group_of(u))) & 1 ? x : 0;
    };
    auto scale_of = [&](uint32_t x, int j, int u) {
        return RT == 16 ? __builtin_amdgcn_readlane((int)x, 4 * j + u) : __shfl((int)x, 4 * j + (ql >> 2), 64);
    };
    const PagedRule<HI> rule(g);
    int64_t M = INT64_MIN;
    if constexpr (PHASE < 2) {
        Score mx = LOW;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (!mine(j)) continue;
            const bool whole_block = all(j);
#pragma unroll
            for (int u = 0; u < TU; u++) {
                const int m = scale_of(mul, j, u), k = whole_block ? 4 : seen(j, u);
                if constexpr (PHASE == 1 && KEEP) {
                    Score x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] = e < k ? (Score)rule.score(D[j][u][e], m) : LOW;
                        mx = x[e] > mx ? x[e] : mx;
                    }
                    if (row < live) {
                        if constexpr (HI) {
                            *(v4i *)kept(j, u) = v4i{(int)x[0], (int)x[1], (int)x[2], (int)x[3]};
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; e++) kept(j, u)[e] = x[e];
                        }
                    }
                    continue;
                }
                int32_t d = INT32_MIN;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int32_t x = e < k ? D[j][u][e] : INT32_MIN;
                    d = x > d ? x : d;
                }
                const Score x = (Score)rule.score(d, m);  // the score grows with the dot
                if (k > 0) mx = x > mx ? x : mx;
            }
        }
#pragma unroll
        for (int o = RT == 16 ? 16 : 4; o < 64; o <<= 1) {  // the lanes of the row
            const Score x = __shfl_xor(mx, o, 64);
            mx = x > mx ? x : mx;
        }
        if (lane < RT) s_mx[w * RT + lane] = mx == LOW ? INT64_MIN : (int64_t)mx;
        if (PHASE == 0 && !mine(0)) wait_vmcnt<0>();  // (no K to wait for)
        lds_barrier();                                // not the fence of __syncthreads, which would wait for V too
        if constexpr (PHASE == 1) {
            if (tid < RT) {
#pragma unroll
                for (int i = 0; i < NW; i++) M = s_mx[i * RT + tid] > M ? s_mx[i * RT + tid] : M;
                S.mx[(slot + range) * RT + tid] = M;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < NW; i++) M = s_mx[i * RT + row] > M ? s_mx[i * RT + row] : M;
    } else if constexpr (DOTS) {
        for (int i = 0; i < ranges; i++) {
            const int64_t x = S.mx[(slot + i) * RT + row];
            M = x > M ? x : M;
        }
        if (!mine(0)) wait_vmcnt<0>();
        if (in_lds) lds_barrier();
    }
    // the entries, in place of the dots
    const int64_t c0 = rule.constant(M == INT64_MIN ? 0 : M);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (!DOTS || !mine(j)) continue;
        const bool whole_block = all(j);
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int m = scale_of(mul, j, u);
#pragma unroll
            for (int e = 0; e < 4; e++) D[j][u][e] = (int32_t)rule.index(D[j][u][e], m, c0, last);
        }
        if (in_lds) {
#pragma unroll
            for (int u = 0; u < TU; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) D[j][u][e] = s_exp[D[j][u][e]];
        } else if (row < live) {
#pragma unroll
            for (int u = 0; u < TU; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) D[j][u][e] = g.exp_table[D[j][u][e]];
        }
        if (!whole_block) {
#pragma unroll
            for (int u = 0; u < TU; u++) {
                const int k = seen(j, u);
#pragma unroll
                for (int e = 0; e < 4; e++) D[j][u][e] = e < k ? D[j][u][e] : 0;
            }
        }
    }
    if constexpr (PHASE != 3) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (!mine(j)) continue;
#pragma unroll
            for (int u = 0; u < TU; u++)  // (entries are below 2^31: a pair sums in 32 bits)
                sum += (uint64_t)((uint32_t)D[j][u][0] + (uint32_t)D[j][u][1]) + ((uint32_t)D[j][u][2] + (uint32_t)D[j][u][3]);
        }
#pragma unroll
        for (int o = RT == 16 ? 16 : 4; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
        if (lane < RT) s_sum[w * RT + lane] = sum;
        lds_barrier();
        if constexpr (PHASE == 2) {
            if (tid < RT) {
                sum = 0;
#pragma unroll
                for (int i = 0; i < NW; i++) sum += s_sum[i * RT + tid];
                S.sum[(place * pl.chunks + range) * RT + tid] = sum;
            }
            return;
        }
        sum = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) sum += s_sum[i * RT + row];
    } else {
        const int sums = KEEP ? (keys + PG_CHUNK - 1) / PG_CHUNK : ranges;
        for (int i = 0; i < sums; i++) sum += S.sum[(place * pl.chunks + i) * RT + row];
        lds_barrier();  // every wave has its entries
    }
    for (int i = tid; i < QC * RT * PG_ACC; i += 64 * NW) s_acc[i] = 0;

    // The digits of w = floor(E 2^P / S) for E = e vs, exactly (softmax_p_of, which holds for E < 2^53 with w <= 2^30), with
    // 0x80808080 inside the rounding constant: the low word of the sum is w + 0x80808080, whose bytes xor 0x80 are
    // balanced digits. D[j][k] word t: digit k of group t's keys (16 rows); D[j][0] word t: digit l % 4 of row l / 4 % 4
    // of group t's keys (4 rows: the lanes transpose through LDS).
    {
        constexpr double magic = 6755399441055744.0 + 2155905152.0;  // 1.5 2^52 + 0x80808080
        const double R = sum > 0 && row < live ? ldexp(1.0 / (double)sum, g.softmax_p) : 0.0, sp = softmax_sp(sum, g.softmax_p);
#pragma unroll
        for (int j = 0; j < NB; j++) {
            __builtin_amdgcn_sched_barrier(0);  // (a block at a time: interleaved they spill)
            if (!mine(j)) continue;
            uint32_t o[TU][4];
#pragma unroll
            for (int u = 0; u < TU; u++) {
                const double scale = (double)(uint32_t)scale_of(vs, j, u);
                uint32_t dg[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const double ed = (double)(uint32_t)D[j][u][e] * scale, x = fma(ed, R, magic), r = fma(x - magic, sp, ed);
                    dg[e] = (uint32_t)__double2loint(x) + (uint32_t)(__double2hiint(r) >> 31);
                }
                byte_transpose(dg[0], dg[1], dg[2], dg[3], o[u]);
            }
            if constexpr (RT == 16) {
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int t = 0; t < 4; t++) D[j][k][t] = (int32_t)(o[t][k] ^ 0x80808080u);
            } else {
                // [row][digit][l / 16][group]
                int *to = (int *)s_v + 64 * (ql & 3) + 4 * qg + (ql >> 2);
#pragma unroll
                for (int k = 0; k < 4; k++) to[16 * k] = (int)(o[0][k] ^ 0x80808080u);
                D[j][0] = *(const v4i *)((const int *)s_v + 16 * ql + 4 * qg);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);

    // sum w v: channels 64 c + 16 i + 4 (l / 16) + e of digit k of row l % 16 in acc[k][i][e] (16 rows), of digit l % 4 of row
    // l / 4 % 4 in acc[0][i][e] (4 rows)
#pragma unroll
    for (int c = 0; c < QC; c++) {
        v4i acc[TU][4];
#pragma unroll
        for (int k = 0; k < TU; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[k][i] = zero;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int f = c * NB + j;  // the loads run ahead over the channels
            v4i(&x)[4] = vr[f % KD];
            __builtin_amdgcn_sched_barrier(0);
            if (mine(j)) {
#pragma unroll
                for (int u = 0; u < 4; u++) *(v4i *)(s_v + 1024 * u + 16 * lane) = x[u];
            }
            if (f + KD < QC * NB) v_load((f + KD) % NB, (f + KD) / NB, x);
            if (!mine(j)) continue;
            const int tr_k = ql >> 1, key = 16 * (tr_k >> 2) + 4 * qg + (tr_k & 3);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int8_t *p0 = s_v + (4 * key + (i ^ vsw<4>(key & 15))) * 16 + 8 * (ql & 1);
                const v2i r0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)p0);
                const v2i r1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(p0 + 32 * 64));
                const v4i vf = v4i{r0[0], r0[1], r1[0], r1[1]};
#pragma unroll
                for (int k = 0; k < TU; k++) acc[k][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf, D[j][k], acc[k][i], 0, 0, 0);
            }
        }
        if (c == 0) lds_barrier();  // the zeros
        if (!mine(0)) continue;
        if constexpr (RT == 16) {
            unsigned long long *to = (unsigned long long *)s_acc + (c * RT + ql) * PG_ACC + 4 * qg;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    // (at most 256 keys a wave: a plane's sum is below 2^22, two planes' below 2^31)
                    const int32_t lo = acc[0][i][e] + acc[1][i][e] * 256, hi = acc[2][i][e] + acc[3][i][e] * 256;
                    atomicAdd(to + 16 * i + e, (unsigned long long)((int64_t)hi * 65536 + lo));
                }
        } else {
            // lane l % 4 = i keeps the four planes' sum of channels 16 i ..: the quad's lanes exchange halves twice
            const bool b0 = lane & 1, b1 = lane & 2;
            int64_t y[2][4], z[4];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int32_t keep = b0 ? acc[0][2 * i + 1][e] : acc[0][2 * i][e], give = b0 ? acc[0][2 * i][e] : acc[0][2 * i + 1][e];
                    const int32_t got = dpp_mov<0xB1>(give);  // of the plane next to this lane's
                    y[i][e] = b0 ? (int64_t)keep * 256 + got : (int64_t)got * 256 + keep;
                }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int64_t keep = b1 ? y[1][e] : y[0][e], got = lane_move64<1>(b1 ? y[0][e] : y[1][e]);
                z[e] = b1 ? keep * 65536 + got : got * 65536 + keep;
            }
            unsigned long long *to = (unsigned long long *)s_acc + (c * RT + (ql >> 2)) * PG_ACC + 16 * (lane & 3) + 4 * qg;
            if ((ql >> 2) < live) {
#pragma unroll
                for (int e = 0; e < 4; e++) atomicAdd(to + e, (unsigned long long)z[e]);
            }
        }
    }
    lds_barrier();
    const double mo = g.out_s > 95 ? 0.0 : ldexp((double)g.out_m, -g.out_s);
    for (int i = tid; i < live * (hd / 4); i += 64 * NW) {
        const int r = i / (hd / 4), ch = 4 * (i - r * (hd / 4));
        const int64_t *x = s_acc + ((ch >> 6) * RT + r) * PG_ACC + (ch & 63);
        if constexpr (PHASE == 3) {
            int64_t *to = S.part + ((slot + range) * RT + r) * hd + ch;
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = x[e];
        } else {
            uint32_t packed = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) packed |= (uint32_t)(uint8_t)(int8_t)attn_out_byte(x[e], mo, g.out_m, g.out_s) << (8 * e);
            const int tok = (row0 + r) / pl.group, head = h * pl.group + (row0 + r) % pl.group;
            *(uint32_t *)(g.out + ((first + tok) * g.heads + head) * hd + ch) = packed;
        }
    }
}

// The scores of a row over PG_CHUNK keys to their entries, in place, and the entries' sum.
template <bool HI>
__global__ __launch_bounds__(256) void k_paged_entries(PagedArgs g, PagedPlan pl, void *scratch) {
    typedef typename std::conditional<HI, int32_t, int64_t>::type Score;
    constexpr Score LOW = HI ? (Score)INT32_MIN : (Score)INT64_MIN;
    constexpr int N = PG_CHUNK / 256;
    __shared__ uint64_t s_sum[4];
    const PagePool &p = g.pages;
    const int tid = threadIdx.x;
    // (row fastest, then the chunk)
    const int r = blockIdx.x % pl.rows, chunk = blockIdx.x / pl.rows % pl.chunks;
    const size_t place = blockIdx.x / pl.rows / pl.chunks;
    const int tile = (int)(place % pl.tiles), s = (int)(place / pl.tiles) / p.kv_heads;
    const int n = (int)(g.ctx[s] < (uint32_t)g.keys ? g.ctx[s] : (uint32_t)g.keys);
    uint32_t count = g.rows ? g.rows[s] : (uint32_t)g.t;
    count = count < (uint32_t)g.t ? count : (uint32_t)g.t;
    const int rows = (int)count * pl.group, row0 = pl.rt * tile, live = rows - row0 < pl.rt ? rows - row0 : pl.rt;
    if (r >= live) return;
    const int keys = n - (int)count + (row0 + live - 1) / pl.group + 1;  // of the tile: those have scores, in whole blocks
    const int k0 = chunk * PG_CHUNK, k1 = (keys + 63) / 64 * 64 < k0 + PG_CHUNK ? (keys + 63) / 64 * 64 : k0 + PG_CHUNK;
    if (k0 >= keys) return;
    const PagedScratch S = paged_scratch(scratch, pl, p.hd);
    Score *at = (Score *)S.keep + (place * pl.rows + r) * ((size_t)pl.ng * pl.span);
    Score x[N];
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        const int key = k0 + 1024 * i + 4 * tid;
        if constexpr (HI) {
            const v4i y = key < k1 ? *(const v4i *)(at + key) : v4i{LOW, LOW, LOW, LOW};
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * i + e] = y[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * i + e] = key < k1 ? at[key + e] : LOW;
        }
    }
    const int ranges = (keys + pl.span - 1) / pl.span;
    int64_t M = INT64_MIN;
    for (int i = tid & 63; i < ranges; i += 64) {
        const int64_t y = S.mx[(place * pl.ng + i) * pl.rt + r];
        M = y > M ? y : M;
    }
    M = wave_max64(M);
    const uint32_t last = (uint32_t)g.exp_len - 1;
    uint64_t sum = 0;
    int32_t y[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint32_t d;
        if constexpr (HI) d = (uint32_t)((int32_t)M - x[i]);
        else d = (uint64_t)(M - x[i]) < last ? (uint32_t)(M - x[i]) : last;
        y[i] = x[i] == LOW ? 0 : g.exp_table[d < last ? d : last];
    }
#pragma unroll
    for (int i = 0; i < N; i++) sum += (uint32_t)y[i];
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        const int key = k0 + 1024 * i + 4 * tid;
        if (key >= k1) continue;
        if constexpr (HI) {
            *(v4i *)(at + key) = v4i{y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) at[key + e] = y[4 * i + e];
        }
    }
    sum = wave_sum_dpp(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) S.sum[(place * pl.chunks + chunk) * pl.rt + r] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
}

// The outputs from the ranges' sums: a thread per four channels.
__global__ __launch_bounds__(256) void k_paged_out(PagedArgs g, PagedPlan pl, void *scratch) {
    const PagePool &p = g.pages;
    const int quads = p.hd / 4;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, at = i / quads;  // (tile of a panel, row)
    const int ch = 4 * (int)(i - at * quads), r = (int)(at % pl.rt);
    const size_t tiles = at / pl.rt;
    if (tiles >= (size_t)pl.panels * pl.tiles) return;
    const int tile = (int)(tiles % pl.tiles), panel = (int)(tiles / pl.tiles), s = panel / p.kv_heads, h = panel - s * p.kv_heads;
    const int n = (int)(g.ctx[s] < (uint32_t)g.keys ? g.ctx[s] : (uint32_t)g.keys);
    uint32_t count = g.rows ? g.rows[s] : (uint32_t)g.t;
    count = count < (uint32_t)g.t ? count : (uint32_t)g.t;
    const int rows = (int)count * pl.group, row0 = pl.rt * tile;
    if (row0 + r >= rows) return;
    const int end = rows - row0 < pl.rt ? rows - row0 : pl.rt;
    const int keys = n - (int)count + (row0 + end - 1) / pl.group + 1;
    const int ranges = keys > pl.span ? (keys + pl.span - 1) / pl.span : 1;
    const PagedScratch S = paged_scratch(scratch, pl, p.hd);
    int64_t x[4] = {0, 0, 0, 0};
    const int64_t *from = S.part + (tiles * pl.ng * pl.rt + r) * p.hd + ch;
    for (int c0 = 0; c0 < ranges; c0 += 8) {  // eight in flight
        int64_t y[8][4];
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) y[c][e] = from[(size_t)(c0 + c < ranges ? c0 + c : c0) * pl.rt * p.hd + e];
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] += c0 + c < ranges ? y[c][e] : 0;
    }
    const double mo = g.out_s > 95 ? 0.0 : ldexp((double)g.out_m, -g.out_s);
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) packed |= (uint32_t)(uint8_t)(int8_t)attn_out_byte(x[e], mo, g.out_m, g.out_s) << (8 * e);
    const int tok = (row0 + r) / pl.group, head = h * pl.group + (row0 + r) % pl.group;
    *(uint32_t *)(g.out + (((size_t)s * g.t + tok) * g.heads + head) * p.hd + ch) = packed;
}

constexpr size_t PG_KEEP = (size_t)128 << 20;  // bytes of scores that a call keeps at most (tiles of 16 rows)

static PagedPlan paged_plan(const PagedArgs &g) {
    PagedPlan p;
    p.group = g.heads / g.pages.kv_heads;
    const long long rows = (long long)g.t * p.group;
    p.rt = rows <= 4 ? 4 : 16;
    p.rows = rows < p.rt ? (int)rows : p.rt;
    p.tiles = (int)((rows + p.rt - 1) / p.rt);
    p.panels = g.streams * g.pages.kv_heads;
    while (1 << p.page_log < g.pages.page) p.page_log++;
    const int most = p.rt == 4 ? 4096 : 2048;  // keys of a tile in one launch
    p.span = (g.keys + 63) / 64 * 64;
    if (g.keys > most) {
        const long long wgs = (long long)p.panels * p.tiles;
        long long ng = (1024 + wgs - 1) / wgs;
        const long long least = (g.keys + 1023) / 1024, more = (g.keys + 255) / 256;  // of 1,024 keys, of 256
        ng = ng < least ? least : (ng > more ? more : ng);
        p.span = (int)(((g.keys + ng - 1) / ng + 255) / 256) * 256;
        p.ng = (g.keys + p.span - 1) / p.span;
        p.store = p.rt == 4 || (size_t)wgs * p.rows * p.ng * p.span * 8 <= PG_KEEP;
        p.chunks = p.store ? (g.keys + PG_CHUNK - 1) / PG_CHUNK : p.ng;
    }
    return p;
}

bool paged_fits(const PagedArgs &g) {
    const PagedPlan p = paged_plan(g);
    return ((long long)p.panels + 7) * p.tiles < (1ll << 23) / p.ng && (long long)p.panels * p.tiles * p.rows < (1ll << 23) / p.chunks && (long long)p.panels * p.tiles * p.rt < (1ll << 31) / (g.pages.hd / 4);
}

size_t paged_workspace(const PagedArgs &g) {
    const PagedPlan p = paged_plan(g);
    size_t bytes = 0;
    if (p.ng > 1) paged_scratch(nullptr, p, g.pages.hd, &bytes);
    return bytes;
}

template <int RT, int QC, int NB, int NW, bool HI, int PHASE, bool KEEP = false>
static hipError_t launch_paged_t(const PagedArgs &g, const PagedPlan &p, void *scratch, hipStream_t stream) {
    const int acc = (8 * QC * RT * PG_ACC + 1023) / 1024 * 1024;
    const int table = RT == 16 && PHASE != 1 && !(KEEP && PHASE == 3) && g.table_lds ? 1024 * ((g.exp_len + 255) / 256) : 0;
    const size_t lds = (size_t)(table > acc ? table : acc) + 4096 * NW + 16 * NW * RT;
    const hipError_t e = allow_dynamic_lds((const void *)k_paged_tile<RT, QC, NB, NW, HI, PHASE, KEEP>, lds);
    if (e != hipSuccess) return e;
    launch_k((k_paged_tile<RT, QC, NB, NW, HI, PHASE, KEEP>), dim3((unsigned)((p.panels + 7) / 8 * 8) * p.tiles * p.ng), dim3(64 * NW), lds, stream, g, p, scratch);
    return hipGetLastError();
}

template <int RT, int QC, bool HI>
static hipError_t launch_paged_q(const PagedArgs &g, const PagedPlan &p, void *scratch, hipStream_t stream) {
    if (p.ng > 1) {
        hipError_t e;
        if (p.store) {
            if ((e = launch_paged_t<RT, QC, 4, 4, HI, 1, true>(g, p, scratch, stream)) != hipSuccess) return e;
            launch_k(k_paged_entries<HI>, dim3((unsigned)p.panels * p.tiles * p.chunks * p.rows), dim3(256), 0, stream, g, p, scratch);
            if ((e = hipGetLastError()) != hipSuccess) return e;
            if ((e = launch_paged_t<RT, QC, 4, 4, HI, 3, true>(g, p, scratch, stream)) != hipSuccess) return e;
        } else if constexpr (RT == 16) {
            if ((e = launch_paged_t<RT, QC, 4, 4, HI, 1>(g, p, scratch, stream)) != hipSuccess) return e;
            if ((e = launch_paged_t<RT, QC, 4, 4, HI, 2>(g, p, scratch, stream)) != hipSuccess) return e;
            if ((e = launch_paged_t<RT, QC, 4, 4, HI, 3>(g, p, scratch, stream)) != hipSuccess) return e;
        }
        const size_t quads = (size_t)p.panels * p.tiles * p.rt * (g.pages.hd / 4);
        launch_k(k_paged_out, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, g, p, scratch);
        return hipGetLastError();
    }
    if (p.span <= 256) return launch_paged_t<RT, QC, 1, 4, HI, 0>(g, p, scratch, stream);
    if (p.span <= 1024) return launch_paged_t<RT, QC, 4, 4, HI, 0>(g, p, scratch, stream);
    if (p.span <= 2048) return launch_paged_t<RT, QC, 4, 8, HI, 0>(g, p, scratch, stream);
    if constexpr (RT == 4) return launch_paged_t<RT, QC, 8, 8, HI, 0>(g, p, scratch, stream);
    return hipErrorInvalidValue;
}

template <int RT>
static hipError_t launch_paged_r(const PagedArgs &g, const PagedPlan &p, void *scratch, hipStream_t stream) {
    const bool hi = g.score_s >= 32 && g.score_s <= 60;
    if (g.pages.hd <= 64) return hi ? launch_paged_q<RT, 1, true>(g, p, scratch, stream) : launch_paged_q<RT, 1, false>(g, p, scratch, stream);
    if (g.pages.hd <= 128) return hi ? launch_paged_q<RT, 2, true>(g, p, scratch, stream) : launch_paged_q<RT, 2, false>(g, p, scratch, stream);
    return hi ? launch_paged_q<RT, 4, true>(g, p, scratch, stream) : launch_paged_q<RT, 4, false>(g, p, scratch, stream);
}

hipError_t launch_paged(const PagedArgs &args, void *workspace, hipStream_t stream) {
    PagedArgs g = args;
    g.table_lds = g.exp_len <= PG_TABLE && (uintptr_t)g.exp_table % 16 == 0;
    const PagedPlan p = paged_plan(g);
    return p.rt == 4 ? launch_paged_r<4>(g, p, workspace, stream) : launch_paged_r<16>(g, p, workspace, stream);
}

}  // namespace hs
