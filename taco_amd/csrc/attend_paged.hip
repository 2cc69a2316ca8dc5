// Attention over pages of 8-bit keys and values with a scale for each page and head (no counterpart in the
// reference): score_j = clamp(rescale(q k_j, score_m ks, score_s), +-2^40), e_j = table[min(M - score_j, len - 1)],
// S = sum e_j, w_j = floor(e_j vs 2^P / S), out = clamp(rescale(sum w_j v_j, out_m, out_s), +-127), with ks and vs the
// scales of key j's page: the rule of the other attention kernels where the scales are 1.
#include "attend.h"

namespace hs {

constexpr int PG_TABLE = 16384;  // entries of the table copied to LDS at most
constexpr int PG_ACC = 66;       // 64 channels' sums of a row and two of padding (bank spread)
constexpr int PG_NONE = 0x7fffffff;  // a lane's offset past any page: the buffer load gives zeros

// n / d without a division: m = ceil(2^32 / d) makes the high word of n m the quotient or one more.
struct PagedDiv {
    uint32_t d = 1, m = 0;
    PagedDiv() = default;
    explicit PagedDiv(uint32_t n) : d(n), m(n > 1 ? 0xffffffffu / n + 1 : 0) {}
    __device__ __forceinline__ int of(int n) const {
        const uint32_t q = m ? __umulhi((uint32_t)n, m) : (uint32_t)n;
        return (int)(q * d > (uint32_t)n ? q - 1 : q);
    }
};

struct PagedPlan {
    int rt = 16;               // rows of a tile
    int group = 1, tiles = 1;  // query heads of a cache head; row tiles of a panel
    int panels = 0;            // (stream, cache head)
    int ng = 1, span = 0;      // key ranges, their keys
    int split = 0;             // several launches, which meet in the scratch
    int store = 0;             // the scores of the ranges are kept there
    int rows = 0, chunks = 1;  // rows of a tile with scores there; of PG_CHUNK keys, with a sum each
    int page_log = 4;
    PagedDiv by_group, by_tiles, by_heads, by_inner;  // group, tiles, cache heads, 8 tiles ng
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

// The table to LDS: whole KiB straight, the rest entry by entry (places past it repeat the last one). The caller waits: the straight
// loads are no LDS operations to a barrier, so each wave waits for its own (table_there, or for loads issued after them).
__device__ __forceinline__ void paged_table(const PagedArgs &g, int32_t *s_exp, int w, int waves, int lane) {
    w = __builtin_amdgcn_readfirstlane(w);
    for (int ch = w; ch < g.exp_len / 256; ch += waves)
        __builtin_amdgcn_global_load_lds((const void *)(g.exp_table + ch * 256 + 4 * lane), (lds_void *)(s_exp + ch * 256), 16, 0, 0);
    if (w == 0)
        for (int i = g.exp_len / 256 * 256 + lane; i < (g.exp_len + 255) / 256 * 256; i += 64)
            s_exp[i] = g.exp_table[i < g.exp_len ? i : g.exp_len - 1];
}

// The tile and key range of a workgroup. Workgroup L runs on XCD L % 8: the tiles of a panel stay on one XCD and share K and V in
// its L2.
struct PagedTile {
    int s, h, tile, range, panel;
    int row0, live;        // its first row, of those that are there
    int before;            // token i of the stream sees keys up to before + i
    int whole, keys;       // the keys that its first row sees, its last
    size_t place, slot;    // of the tile, of its ranges in the scratch
    bool there;
    __device__ __forceinline__ PagedTile() {}
    __device__ __forceinline__ PagedTile(const PagedArgs &g, const PagedPlan &pl, int L) {
        const int inner = pl.tiles * pl.ng, group = pl.by_inner.of(L);
        panel = 8 * group + (L & 7);
        const int in = (L - 8 * inner * group) >> 3;
        range = pl.by_tiles.of(in);
        tile = in - range * pl.tiles;
        there = panel < pl.panels;
        if (!there) return;
        s = pl.by_heads.of(panel);
        h = panel - s * g.pages.kv_heads;
        place = (size_t)panel * pl.tiles + tile;
        slot = place * pl.ng;
    }
    // with the stream's counts
    __device__ __forceinline__ void rows(const PagedArgs &g, const PagedPlan &pl, uint32_t ctx, uint32_t count) {
        const int n = (int)(ctx < (uint32_t)g.keys ? ctx : (uint32_t)g.keys);
        count = count < (uint32_t)g.t ? count : (uint32_t)g.t;
        const int all = (int)count * pl.group;
        row0 = pl.rt * tile;
        live = all - row0 < pl.rt ? all - row0 : pl.rt;
        before = n - (int)count;
        whole = before + pl.by_group.of(row0) + 1;
        keys = live > 0 ? before + pl.by_group.of(row0 + live - 1) + 1 : 0;
    }
};

// The pages of a wave's blocks of 64 keys (the wave's block j starts at key first + step j, at most 16 of them): lane 4 j + t
// knows the page of group t, the 16 keys from 16 t on.
struct PagedBlocks {
    uint32_t number;
    uint32_t at_lo, at_hi;  // where the group's rows start in the pools
    uint64_t there;         // the groups with keys and a page
    int first, step;
    // (before the stream's counts are known: entries up to `keys` are there for every stream)
    __device__ __forceinline__ PagedBlocks(const PagedArgs &g, const PagedPlan &pl, int s, int k0, int st, int blocks, int lane) : first(k0), step(st) {
        const int key = key_of(lane >> 2) + 16 * (lane & 3);
        number = 0xffffffffu;
        if ((lane >> 2) < blocks && key < g.keys) number = g.table[(size_t)s * g.width + (key >> pl.page_log)];
    }
    __device__ __forceinline__ void until(const PagedArgs &g, const PagedPlan &pl, int h, int k1, int lane) {
        const PagePool &p = g.pages;
        const int key = key_of(lane >> 2) + 16 * (lane & 3);
        if (key >= k1) number = 0xffffffffu;
        there = __ballot(number < (uint32_t)p.pages);
        const uint64_t row = (((uint64_t)number * (uint32_t)p.kv_heads + h) << pl.page_log) + (key & (p.page - 1));
        const uint64_t at = row * (uint32_t)p.hd;
        at_lo = (uint32_t)at;
        at_hi = (uint32_t)(at >> 32);
    }
    __device__ __forceinline__ int key_of(int j) const { return first + step * j; }
    __device__ __forceinline__ bool has(int j, int t) const { return (there >> (4 * j + t)) & 1; }
    // this lane's page's scale, 1 ..= max_scale (1 without a page)
    __device__ __forceinline__ uint32_t scale(const PagedArgs &g, const uint32_t *scales, int h) const {
        uint32_t x = 1;
        if (number < (uint32_t)g.pages.pages) x = scales[(size_t)number * g.pages.kv_heads + h];
        return x < 1 ? 1 : (x > g.pages.max_scale ? g.pages.max_scale : x);
    }
    // the 16 rows of a group; loads of one that is not there give zeros without an access
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(const PagedArgs &g, const int8_t *pool, int j, int t) const {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)at_lo, 4 * j + t), hi = (uint32_t)__builtin_amdgcn_readlane((int)at_hi, 4 * j + t);
        return __builtin_amdgcn_make_buffer_rsrc((void *)(pool + ((uint64_t)hi << 32 | lo)), 0, has(j, t) ? 16 * g.pages.hd : 0, 0x00020000);
    }
};
__device__ __forceinline__ v4i paged_load(__amdgpu_buffer_rsrc_t r, int at) {
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}
// K as the product's operand (chunk c: bytes 64 c + 16 (l / 16) .. of row l % 16); channels past the head are zeros
template <int QC>
__device__ __forceinline__ void paged_k(const PagedArgs &g, const PagedBlocks &b, int j, int lane, v4i (&x)[4][QC]) {
    const int hd = g.pages.hd;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const auto r = b.rows(g, g.pages.k, j, t);
#pragma unroll
        for (int c = 0; c < QC; c++) {
            const int o = 64 * c + 16 * (lane >> 4);
            x[t][c] = paged_load(r, o < hd ? (lane & 15) * hd + o : PG_NONE);
        }
    }
}
// 64 channels of V for paged_pv: lane l has 16-byte chunk l % 4, swizzled, of row l / 4 of each group
__device__ __forceinline__ void paged_v(const PagedArgs &g, const PagedBlocks &b, int j, int c, int lane, v4i (&x)[4]) {
    const int hd = g.pages.hd, r = lane >> 2, o = 64 * c + 16 * ((lane & 3) ^ vsw<4>(r)), at = o < hd ? r * hd + o : PG_NONE;
#pragma unroll
    for (int t = 0; t < 4; t++) x[t] = paged_load(b.rows(g, g.pages.v, j, t), at);
}
// q of a tile's rows from row r0 on as the product's operand: operand t has row r in column RT t + r.
template <int RT, int QC>
__device__ __forceinline__ void paged_q(const PagedArgs &g, const PagedPlan &pl, const PagedTile &T, int r0, int lane, v4i (&q)[16 / RT][QC]) {
    const int ql = lane & 15, row = r0 + ql % RT, tok = pl.by_group.of(T.row0 + row);
    const int head = T.h * pl.group + T.row0 + row - tok * pl.group;
    const v4i zero = v4i{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < QC; c++) {
        const int o = 64 * c + 16 * (lane >> 4);
        const v4i x = row < T.live && o < g.pages.hd
                          ? *(const v4i *)(g.q + ((size_t)T.s * g.t + tok) * g.q_stride + (size_t)head * g.pages.hd + o) : zero;
        if constexpr (RT == 16) {
            q[0][c] = x;
        } else {
#pragma unroll
            for (int t = 0; t < 16 / RT; t++) q[t][c] = ql / RT == t ? x : zero;
        }
    }
}
// The dots of a block.
template <int RT, int QC>
__device__ __forceinline__ void paged_dots(const v4i (&x)[4][QC], const v4i (&q)[16 / RT][QC], v4i (&D)[RT / 4]) {
    constexpr int G = 16 / RT;  // groups in an accumulator
#pragma unroll
    for (int u = 0; u < RT / 4; u++) D[u] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int c = 0; c < QC; c++) {
            v4i &d = D[t / G];
            d = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[t][c], q[t % G][c], d, 0, 0, 0);
        }
}
// Of a value that lane 4 j + t holds, that of this lane's group of accumulator u.
template <int RT>
__device__ __forceinline__ int paged_of(uint32_t x, int j, int u, int lane) {
    return RT == 16 ? __builtin_amdgcn_readlane((int)x, 4 * j + u) : __shfl((int)x, 4 * j + 16 / RT * u + (lane & 15) / RT, 64);
}

// The digits of w = floor(E 2^P / S) for E = e vs, exactly (softmax_p_of, which holds for E < 2^53 with w <= 2^30), with
// 0x80808080 inside the rounding constant: the low word of the sum is w + 0x80808080, whose bytes xor 0x80 are balanced
// digits. From the entries D[u][e]: D[k] word t the digit k of group t's keys (16 rows); D[0] word t digit l % 4 of row
// l / 4 % 4 of group t's keys (4 rows), D[k] word t digit 2 k + l % 2 of row l / 2 % 8 (8 rows): the lanes transpose through
// 256 bytes of LDS a row.
struct PagedWeight {
    double R, sp;  // rows that are not there and rows without weight: w = 0 (R = 0)
    __device__ __forceinline__ PagedWeight(uint64_t sum, int P, bool live)
        : R(sum > 0 && live ? ldexp(1.0 / (double)sum, P) : 0.0), sp(softmax_sp(sum, P)) {}
};
template <int RT>
__device__ __forceinline__ void paged_digits(const PagedWeight &wt, uint32_t vs, int j, int lane, int8_t *mem, v4i (&D)[RT / 4]) {
    constexpr double magic = 6755399441055744.0 + 2155905152.0;  // 1.5 2^52 + 0x80808080
    constexpr int TU = RT / 4;
    const int ql = lane & 15, qg = lane >> 4;
    uint32_t o[TU][4];
#pragma unroll
    for (int u = 0; u < TU; u++) {
        const double scale = (double)(uint32_t)paged_of<RT>(vs, j, u, lane);
        uint32_t dg[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double ed = (double)(uint32_t)D[u][e] * scale, x = fma(ed, wt.R, magic), r = fma(x - magic, wt.sp, ed);
            dg[e] = (uint32_t)__double2loint(x) + (uint32_t)(__double2hiint(r) >> 31);
        }
        byte_transpose(dg[0], dg[1], dg[2], dg[3], o[u]);
        if (RT == 16) __builtin_amdgcn_sched_barrier(0);  // (interleaved they spill)
    }
    if constexpr (RT == 16) {
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int t = 0; t < 4; t++) D[k][t] = (int32_t)(o[t][k] ^ 0x80808080u);
    } else {
        int *to = (int *)mem + 64 * (ql % RT) + 4 * qg + ql / RT;  // [row][digit][l / 16][group]
#pragma unroll
        for (int u = 0; u < TU; u++)
#pragma unroll
            for (int k = 0; k < 4; k++) to[16 * k + 16 / RT * u] = (int)(o[u][k] ^ 0x80808080u);
#pragma unroll
        for (int k = 0; k < TU; k++) D[k] = *(const v4i *)((const int *)mem + 64 * (ql / (4 / TU)) + 16 * (4 / TU * k + ql % (4 / TU)) + 4 * qg);
    }
}
// acc += V^T digits over a block, 64 channels of V through 4 KiB of LDS: channels 16 i + 4 (l / 16) + e of digit k of row l % 16
// in acc[k][i][e] (16 rows), of the digit and row of D[k] as above (4 and 8).
// `then` runs when x has left the registers.
template <int RT, typename F>
__device__ __forceinline__ void paged_pv(const v4i (&x)[4], const v4i (&D)[RT / 4], int lane, int8_t *mem, v4i (&acc)[RT / 4][4], F then) {
    const int ql = lane & 15, qg = lane >> 4, tr_k = ql >> 1, key = 16 * (tr_k >> 2) + 4 * qg + (tr_k & 3);
#pragma unroll
    for (int u = 0; u < 4; u++) *(v4i *)(mem + 1024 * u + 16 * lane) = x[u];
    then();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int8_t *p0 = mem + (4 * key + (i ^ vsw<4>(key & 15))) * 16 + 8 * (ql & 1);
        const v2i r0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)p0);
        const v2i r1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(p0 + 32 * 64));
        const v4i vf = v4i{r0[0], r0[1], r1[0], r1[1]};
#pragma unroll
        for (int k = 0; k < RT / 4; k++) acc[k][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf, D[k], acc[k][i], 0, 0, 0);
    }
}
// The planes' sums of 64 channels of a wave added to the rows' sums s_acc[RT][PG_ACC]; SMALL: at most 256 keys, two planes' sums
// below 2^31.
template <int RT, bool SMALL>
__device__ __forceinline__ void paged_add(const v4i (&acc)[RT / 4][4], int live, int lane, int64_t *s_acc) {
    const int ql = lane & 15, qg = lane >> 4;
    if constexpr (RT == 16) {
        unsigned long long *to = (unsigned long long *)s_acc + ql * PG_ACC + 4 * qg;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                int64_t x;
                if constexpr (SMALL) {
                    const int32_t lo = acc[0][i][e] + acc[1][i][e] * 256, hi = acc[2][i][e] + acc[3][i][e] * 256;
                    x = (int64_t)hi * 65536 + lo;
                } else {
                    const int64_t lo = (int64_t)acc[1][i][e] * 256 + acc[0][i][e], hi = (int64_t)acc[3][i][e] * 256 + acc[2][i][e];
                    x = hi * 65536 + lo;
                }
                atomicAdd(to + 16 * i + e, (unsigned long long)x);
            }
    } else if constexpr (RT == 8) {
        // lane l % 2 keeps the four planes' sum of channels 32 (l % 2) ..: the pair's lanes exchange halves
        const bool b = lane & 1;
        unsigned long long *to = (unsigned long long *)s_acc + (ql >> 1) * PG_ACC + 32 * (lane & 1) + 4 * qg;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                int64_t z[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int32_t keep = b ? acc[k][i + 2][e] : acc[k][i][e], got = dpp_mov<0xB1>(b ? acc[k][i][e] : acc[k][i + 2][e]);
                    z[k] = b ? (int64_t)keep * 256 + got : (int64_t)got * 256 + keep;
                }
                if ((ql >> 1) < live) atomicAdd(to + 16 * i + e, (unsigned long long)(z[1] * 65536 + z[0]));
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
        unsigned long long *to = (unsigned long long *)s_acc + (ql >> 2) * PG_ACC + 16 * (lane & 3) + 4 * qg;
        if ((ql >> 2) < live) {
#pragma unroll
            for (int e = 0; e < 4; e++) atomicAdd(to + e, (unsigned long long)z[e]);
        }
    }
}
// Four output bytes of a row.
__device__ __forceinline__ void paged_put(const PagedArgs &g, const PagedPlan &pl, int s, int h, int row, int ch, const int64_t *x) {
    const double mo = g.out_s > 95 ? 0.0 : ldexp((double)g.out_m, -g.out_s);
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) packed |= (uint32_t)(uint8_t)(int8_t)attn_out_byte(x[e], mo, g.out_m, g.out_s) << (8 * e);
    const int tok = pl.by_group.of(row), head = h * pl.group + row - tok * pl.group;
    *(uint32_t *)(g.out + (((size_t)s * g.t + tok) * g.heads + head) * g.pages.hd + ch) = packed;
}

// Tiles of RT rows (16, or 4 or 8 where there are no more) of one (stream, cache head): row r is query head r % group of
// token r / group. Wave w takes the blocks of 64 keys w, w + NW, .. of the range, NB at most, each in four groups of 16
// keys that lie in one page. K is the first operand of v_mfma_i32_16x16x64_i8, so lane l holds dots of column l % 16
// with keys 4 (l / 16) + e of a group. With 16 rows a column is a row and D[t] holds group t. With 4 rows column 4 t + r is
// row r with group t: the products of the four groups add up in one accumulator, each with q in its own columns and
// zeros in the others, so that no lane idles; the product with V takes the rows' four digit planes as its 16 columns. With 8
// rows two groups share an accumulator and two planes a product.
// What bounds it: one row, HBM (768 panels of 64 channels: 512 to 1,024 keys 76 MB in 19.3 us, 4,096 to 8,192 keys 605 MB in 117,
// 5.2 TB/s). Few panels, what one CU reads, some 30 KB a us (12 panels of 4,096 to 8,192 keys 27 us; 128 of 2,000 to 4,000 keys
// with 128 channels and 8 rows 42). Many rows, VALU issue: 192 panels of 256 causal rows over 512 to 1,024 keys, 16.5 M instructions, 27 us of 50.
// A few forms spill registers: one row of up to 16,384 keys 4, of 256 channels 8.
// All in one launch, the dots in registers from the one product to the other: the rule needs the row's largest score and its sum
// before a weight, and forming the dots again would read K again. The table goes to LDS for more than 4 rows; for few rows the
// lookups are fewer than its entries.
template <int RT, int QC, int NB, int NW, bool HI>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW > 8 || (RT <= 8 && NW == 8 && QC <= 2) ? 4 : QC == 1 && RT == 16 ? 3 : 2))) void k_paged_tile(PagedArgs g, PagedPlan pl) {
    static_assert(NB <= 16, "a lane for each group of the wave's blocks");
    static_assert(RT < 16 || NB <= 4, "two planes' sums of a wave's keys in 32 bits");
    constexpr int TU = RT / 4;  // accumulators of a block
    constexpr int KD = QC == 1 && NB <= 8 ? (NB < 2 ? NB : RT >= 8 || NW >= 8 ? 2 : NB < 4 ? NB : 4) : QC == 2 && NB > 1 && NW <= 8 ? 2 : 1;  // blocks of K in flight, and of V
    typedef typename std::conditional<HI, int32_t, int64_t>::type Score;
    constexpr Score LOW = HI ? (Score)INT32_MIN : (Score)INT64_MIN;
    extern __shared__ __attribute__((aligned(1024))) int8_t s_mem[];
    const PagePool &p = g.pages;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4, hd = p.hd;
    PagedTile T(g, pl, blockIdx.x);
    if (!T.there) return;
    const uint32_t ctx = g.ctx[T.s], count = g.rows ? g.rows[T.s] : (uint32_t)g.t;
    PagedBlocks B(g, pl, T.s, 64 * w, 64 * NW, NB, lane);
    T.rows(g, pl, ctx, count);
    if (T.live <= 0) return;
    const int k1 = T.keys;
    const uint32_t last = (uint32_t)g.exp_len - 1;

    // LDS: the table (of more than 4 rows), which the sums of the outputs take over, each wave's V, what the waves exchange
    const bool in_lds = RT >= 8 && g.table_lds;
    constexpr int ACC_BYTES = (8 * QC * RT * PG_ACC + 1023) / 1024 * 1024;
    const int table_bytes = in_lds ? 1024 * ((g.exp_len + 255) / 256) : 0;
    const int top = table_bytes > ACC_BYTES ? table_bytes : ACC_BYTES;
    int32_t *s_exp = (int32_t *)s_mem;
    int64_t *s_acc = (int64_t *)s_mem;  // [QC][RT][PG_ACC]
    int8_t *s_v = s_mem + top + 4096 * w;
    uint64_t *s_sum = (uint64_t *)(s_mem + top + 4096 * NW);  // [NW][RT]
    int64_t *s_mx = (int64_t *)(s_sum + NW * RT);             // [NW][RT]
    if (in_lds) {
        paged_table(g, s_exp, w, NW, lane);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);  // the table's loads before those of K: who has K has the table
    }
    B.until(g, pl, T.h, k1, lane);
    auto mine = [&](int j) { return B.key_of(j) < k1; };  // uniform
    const int row = ql % RT, near = row < T.live ? row : T.live - 1;  // rows that are not there: as the last one
    v4i D[NB][TU], vr[KD][4], qf[16 / RT][QC];
    // all loads without a branch around them, so that the waits count them exactly
    v4i kr[KD][4][QC];
#pragma unroll
    for (int j = 0; j < KD; j++) paged_k<QC>(g, B, j, lane, kr[j]);
    paged_q<RT, QC>(g, pl, T, 0, lane, qf);
    const uint32_t mul = B.scale(g, p.k_scale, T.h) * (uint32_t)g.score_m, vs = B.scale(g, p.v_scale, T.h);
    if constexpr (NB <= KD) {
#pragma unroll
        for (int j = 0; j < NB; j++) paged_v(g, B, j, 0, lane, vr[j]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (mine(j)) paged_dots<RT, QC>(kr[j % KD], qf, D[j]);
        if (j + KD < NB) paged_k<QC>(g, B, j + KD, lane, kr[j % KD]);
        if (NB > 4) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (NB > KD) {
#pragma unroll
        for (int j = 0; j < KD; j++) paged_v(g, B, j, 0, lane, vr[j]);
    }

    // which of a lane's keys its row sees, where not all do
    const int most = T.whole < k1 ? T.whole : k1;
    auto all = [&](int j) { return B.key_of(j) + 64 <= most && ((B.there >> (4 * j)) & 15) == 15; };  // uniform
    const int sees = T.before + pl.by_group.of(T.row0 + near) + 1, lim = sees < k1 ? sees : k1;
    auto seen = [&](int j, int u) {  // how many of the lane's four keys
        const int t = 16 / RT * u + ql / RT;
        return B.has(j, t) ? lim - (B.key_of(j) + 16 * t + 4 * qg) : 0;
    };
    const PagedRule<HI> rule(g);
    Score mx = LOW;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (!mine(j)) continue;
        const bool whole_block = all(j);
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int m = paged_of<RT>(mul, j, u, lane);
            v4i y = D[j][u];
            int k = 4;
            if (!whole_block) {
                k = seen(j, u);
#pragma unroll
                for (int e = 1; e < 4; e++) y[e] = e < k ? y[e] : y[0];  // (with none the result is not used)
            }
            const int32_t a = y[0] > y[1] ? y[0] : y[1], b = y[2] > y[3] ? y[2] : y[3];
            const Score x = (Score)rule.score(a > b ? a : b, m);  // the score grows with the dot
            if (whole_block || k > 0) mx = x > mx ? x : mx;
        }
    }
#pragma unroll
    for (int o = RT; o < 64; o <<= 1) {  // the lanes of the row
        const Score x = __shfl_xor(mx, o, 64);
        mx = x > mx ? x : mx;
    }
    if (lane < RT) s_mx[w * RT + lane] = mx == LOW ? INT64_MIN : (int64_t)mx;
    if (!mine(0)) wait_vmcnt<0>();  // (no K to wait for, whose loads are behind the table's)
    lds_barrier();                  // (V stays in flight)
    int64_t M = INT64_MIN;
#pragma unroll
    for (int i = 0; i < NW; i++) M = s_mx[i * RT + row] > M ? s_mx[i * RT + row] : M;
    // the entries, in place of the dots
    const int64_t c0 = rule.constant(M == INT64_MIN ? 0 : M);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (!mine(j)) continue;
        const bool whole_block = all(j);
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int m = paged_of<RT>(mul, j, u, lane);
#pragma unroll
            for (int e = 0; e < 4; e++) D[j][u][e] = (int32_t)rule.index(D[j][u][e], m, c0, last);
        }
        if (in_lds) {
#pragma unroll
            for (int u = 0; u < TU; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) D[j][u][e] = s_exp[D[j][u][e]];
        } else if (row < T.live) {
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
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (!mine(j)) continue;
#pragma unroll
        for (int u = 0; u < TU; u++)  // (entries are below 2^31: a pair sums in 32 bits)
            sum += (uint64_t)((uint32_t)D[j][u][0] + (uint32_t)D[j][u][1]) + ((uint32_t)D[j][u][2] + (uint32_t)D[j][u][3]);
    }
#pragma unroll
    for (int o = RT; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (lane < RT) s_sum[w * RT + lane] = sum;
    lds_barrier();
    sum = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) sum += s_sum[i * RT + row];
    for (int i = tid; i < QC * RT * PG_ACC; i += 64 * NW) s_acc[i] = 0;
    const PagedWeight wt(sum, g.softmax_p, row < T.live);
#pragma unroll
    for (int j = 0; j < NB; j++) {
        __builtin_amdgcn_sched_barrier(0);  // (a block at a time: interleaved they spill)
        if (mine(j)) paged_digits<RT>(wt, vs, j, lane, s_v, D[j]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < QC; c++) {
        v4i acc[TU][4];
#pragma unroll
        for (int k = 0; k < TU; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[k][i] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int f = c * NB + j;  // the loads run ahead over the channels
            __builtin_amdgcn_sched_barrier(0);
            if (mine(j)) paged_pv<RT>(vr[f % KD], D[j], lane, s_v, acc, [] {});
            if (f + KD < QC * NB) paged_v(g, B, (f + KD) % NB, (f + KD) / NB, lane, vr[f % KD]);
        }
        if (c == 0) lds_barrier();  // the zeros
        if (mine(0)) paged_add<RT, (NB <= 4)>(acc, T.live, lane, s_acc + c * RT * PG_ACC);
    }
    lds_barrier();
    for (int i = tid; i < T.live * (hd / 4); i += 64 * NW) {
        const int r = i / (hd / 4), ch = 4 * (i - r * (hd / 4));
        const int64_t *x = s_acc + ((ch >> 6) * RT + r) * PG_ACC + (ch & 63);
        paged_put(g, pl, T.s, T.h, T.row0 + r, ch, x);
    }
}

// ---- Ranges that leave their scores in the scratch ------------------------------------------------------
// Three launches and a join: the scores of every key (K once), their entries and sums, the products with V (V once). Four waves
// walk a range's blocks, at most 16 each, with the next blocks' loads under way; what a workgroup has to find out first (counts,
// pages, scales) is spread over up to 4,096 keys. For one row the scratch is 8 (i32) of 136 bytes a key; HBM bounds scores and
// products: 200 panels of 8,192 to 16,384 keys (which one launch takes now), 158 MB each, 35 and 38 us (4.5 and 4.1 TB/s), the
// entries between them 8.6, the join 5.
template <int RT, int QC, bool HI>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QC == 4 ? 2 : 4))) void k_paged_scores(PagedArgs g, PagedPlan pl, void *scratch) {
    typedef typename std::conditional<HI, int32_t, int64_t>::type Score;
    constexpr Score LOW = HI ? (Score)INT32_MIN : (Score)INT64_MIN;
    constexpr int TU = RT / 4;
    __shared__ int64_t s_mx[4][RT];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4;
    PagedTile T(g, pl, blockIdx.x);
    if (!T.there) return;
    const int k0 = T.range * pl.span;
    const uint32_t ctx = g.ctx[T.s], count = g.rows ? g.rows[T.s] : (uint32_t)g.t;
    PagedBlocks B(g, pl, T.s, k0 + 64 * w, 256, 16, lane);
    T.rows(g, pl, ctx, count);
    if (T.live <= 0 || k0 >= T.keys) return;  // the launches behind read no result of this range
    const int k1 = k0 + pl.span < T.keys ? k0 + pl.span : T.keys;
    B.until(g, pl, T.h, k1, lane);
    const int row = RT == 16 ? ql : ql & 3, near = row < T.live ? row : T.live - 1;
    const PagedScratch S = paged_scratch(scratch, pl, g.pages.hd);
    constexpr int KD = QC == 1 ? 3 : 2;  // blocks of K in flight, with the one at work
    v4i x[KD][4][QC], qf[16 / RT][QC];
#pragma unroll
    for (int j = 0; j + 1 < KD; j++) paged_k<QC>(g, B, j, lane, x[j]);
    paged_q<RT, QC>(g, pl, T, 0, lane, qf);
    const uint32_t mul = B.scale(g, g.pages.k_scale, T.h) * (uint32_t)g.score_m;
    const int sees = T.before + pl.by_group.of(T.row0 + near) + 1, lim = sees < k1 ? sees : k1, most = T.whole < k1 ? T.whole : k1;
    const PagedRule<HI> rule(g);
    Score mx = LOW;
    Score *to = (Score *)S.keep + (T.place * pl.rows + row) * ((size_t)pl.ng * pl.span) + 4 * qg + (RT == 16 ? 0 : 16 * (ql >> 2));
    auto step = [&](int j, v4i (&now)[4][QC], v4i (&next)[4][QC]) {
        if (j + KD - 1 < 16) paged_k<QC>(g, B, j + KD - 1, lane, next);  // (past the range: no access)
        v4i D[TU];
        paged_dots<RT, QC>(now, qf, D);
        const int key = B.key_of(j);
        const bool whole = key + 64 <= most && ((B.there >> (4 * j)) & 15) == 15;  // uniform
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const int t = RT == 16 ? u : ql >> 2, m = paged_of<RT>(mul, j, u, lane);
            const int k = whole ? 4 : B.has(j, t) ? lim - (key + 16 * t + 4 * qg) : 0;
            Score y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                y[e] = whole || e < k ? (Score)rule.score(D[u][e], m) : LOW;
                mx = y[e] > mx ? y[e] : mx;
            }
            if (row < T.live) {
                Score *at = to + key + (RT == 16 ? 16 * u : 0);
                if constexpr (HI) {
                    *(v4i *)at = v4i{(int)y[0], (int)y[1], (int)y[2], (int)y[3]};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) at[e] = y[e];
                }
            }
        }
        return B.key_of(j + 1) < k1;
    };
    if (B.key_of(0) < k1)
        for (int j = 0;; j += KD) {
            if (!step(j, x[0], x[KD - 1]) || !step(j + 1, x[1], x[0])) break;
            if constexpr (KD == 3)
                if (!step(j + 2, x[2], x[1])) break;
        }
#pragma unroll
    for (int o = RT == 16 ? 16 : 4; o < 64; o <<= 1) {
        const Score y = __shfl_xor(mx, o, 64);
        mx = y > mx ? y : mx;
    }
    if (lane < RT) s_mx[w][lane] = mx == LOW ? INT64_MIN : (int64_t)mx;
    __syncthreads();
    if (tid < RT) {
        int64_t M = s_mx[0][tid];
#pragma unroll
        for (int i = 1; i < 4; i++) M = s_mx[i][tid] > M ? s_mx[i][tid] : M;
        S.mx[(T.slot + T.range) * RT + tid] = M;
    }
}

// GC chunks of 64 channels from chunk GC blockIdx.y on.
template <int RT, int GC, bool HI>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(RT == 16 && GC > 1 ? 2 : 3))) void k_paged_products(PagedArgs g, PagedPlan pl, void *scratch) {
    typedef typename std::conditional<HI, int32_t, int64_t>::type Score;
    constexpr int TU = RT / 4;
    __shared__ __attribute__((aligned(1024))) int8_t s_mem[4][4096];
    __shared__ int64_t s_acc[GC * RT * PG_ACC];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4, hd = g.pages.hd, c0 = GC * blockIdx.y;
    PagedTile T(g, pl, blockIdx.x);
    if (!T.there) return;
    const int k0 = T.range * pl.span;
    const uint32_t ctx = g.ctx[T.s], count = g.rows ? g.rows[T.s] : (uint32_t)g.t;
    PagedBlocks B(g, pl, T.s, k0 + 64 * w, 256, 16, lane);
    for (int i = tid; i < GC * RT * PG_ACC; i += 256) s_acc[i] = 0;
    T.rows(g, pl, ctx, count);
    if (T.live <= 0 || (k0 >= T.keys && T.range > 0)) return;  // the join reads no result of this range
    const int k1 = k0 + pl.span < T.keys ? k0 + pl.span : T.keys;
    B.until(g, pl, T.h, k1, lane);
    const int row = RT == 16 ? ql : ql & 3;
    const bool live = row < T.live;
    const PagedScratch S = paged_scratch(scratch, pl, hd);
    const Score *from = (const Score *)S.keep + (T.place * pl.rows + (live ? row : 0)) * ((size_t)pl.ng * pl.span) + 4 * qg + (RT == 16 ? 0 : 16 * (ql >> 2));
    auto entries = [&](int j, v4i (&D)[TU]) {
        const int key = B.key_of(j) < k1 ? B.key_of(j) : k0;
#pragma unroll
        for (int u = 0; u < TU; u++) {
            const Score *at = from + key + (RT == 16 ? 16 * u : 0);
            if constexpr (HI) {
                D[u] = *(const v4i *)at;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) D[u][e] = (int32_t)at[e];
            }
        }
    };
    v4i x[GC][4], D[TU];
    const bool any = B.key_of(0) < k1;
    if (any) entries(0, D);
#pragma unroll
    for (int c = 0; c < GC; c++) paged_v(g, B, 0, c0 + c, lane, x[c]);
    const uint32_t vs = B.scale(g, g.pages.v_scale, T.h);
    uint64_t sum = 0;
    const int sums = (T.keys + PG_CHUNK - 1) / PG_CHUNK;
    for (int i = 0; i < sums; i++) sum += S.sum[(T.place * pl.chunks + i) * RT + (live ? row : 0)];
    const PagedWeight wt(sum, g.softmax_p, live);
    v4i acc[GC][TU][4];
#pragma unroll
    for (int c = 0; c < GC; c++)
#pragma unroll
        for (int k = 0; k < TU; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[c][k][i] = v4i{0, 0, 0, 0};
    // (one step a turn, the entries copied: with two and an exit between them the sums are held twice and spill)
    for (int j = 0; B.key_of(j) < k1; j++) {
        v4i E[TU];
#pragma unroll
        for (int u = 0; u < TU; u++) E[u] = D[u];
        entries(j + 1, D);
        __builtin_amdgcn_sched_barrier(0);
        paged_digits<RT>(wt, vs, j, lane, s_mem[w], E);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < GC; c++) {
            paged_pv<RT>(x[c], E, lane, s_mem[w], acc[c], [&] {
                __builtin_amdgcn_sched_barrier(0);
                if (j + 1 < 16) paged_v(g, B, j + 1, c0 + c, lane, x[c]);  // (past the range: no access)
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }
    __syncthreads();  // the zeros
    if (any) {
#pragma unroll
        for (int c = 0; c < GC; c++) paged_add<RT, false>(acc[c], T.live, lane, s_acc + c * RT * PG_ACC);
    }
    __syncthreads();
    const int chs = hd - 64 * c0 < 64 * GC ? hd - 64 * c0 : 64 * GC;  // channels here
    for (int i = tid; i < T.live * (chs / 4); i += 256) {
        const int r = i / (chs / 4), ch = 4 * (i - r * (chs / 4));
        const int64_t *y = s_acc + ((ch >> 6) * RT + r) * PG_ACC + (ch & 63);
        int64_t *to = S.part + ((T.slot + T.range) * RT + r) * hd + 64 * c0 + ch;
#pragma unroll
        for (int e = 0; e < 4; e++) to[e] = y[e];
    }
}

// ---- Many rows over long caches ------------------------------------------------------------------------
// Groups of 64 rows, four tiles of 16: three walks over a range's keys, each forming the dots again (4 MFMAs a block and tile,
// less than keeping 16 scores a key and tile would cost): the largest scores, the sums of the entries, the products with V.
// In the first two a wave takes blocks of keys with all four tiles, so that the four waves' loads are of different keys; in
// the third a wave takes a tile over all blocks, since a tile's sums are 64 registers for 64 channels (the waves' loads of
// the same rows meet in the L1). VALU issue bounds them, and few workgroups where there are few panels: 192 panels of 64 rows over
// 2,048 to 4,096 keys 100 us (38 M scores), 12 panels of 256 rows over 16,000 keys 157.
// The second walk spills registers past 64 channels: 21 to 128 channels and 47 to 256, with scores of 64 bits 32 and 67.
template <int QC, bool HI, int PHASE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QC == 4 ? 2 : 3))) void k_paged_scan(PagedArgs g, PagedPlan pl, void *scratch) {
    extern __shared__ __attribute__((aligned(1024))) int32_t s_exp[];  // the table
    __shared__ int64_t s_x[4][64];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4;
    PagedTile T(g, pl, blockIdx.x);
    if (!T.there) return;
    if (PHASE == 2 && g.table_lds) paged_table(g, s_exp, w, 4, lane);
    const int k0 = T.range * pl.span;
    const uint32_t ctx = g.ctx[T.s], count = g.rows ? g.rows[T.s] : (uint32_t)g.t;
    PagedBlocks B(g, pl, T.s, k0 + 64 * w, 256, 16, lane);
    T.rows(g, pl, ctx, count);
    if (T.live <= 0 || k0 >= T.keys) return;  // the launches behind read no result of this range
    const int k1 = k0 + pl.span < T.keys ? k0 + pl.span : T.keys, tiles = (T.live + 15) / 16;
    B.until(g, pl, T.h, k1, lane);
    const PagedScratch S = paged_scratch(scratch, pl, g.pages.hd);
    v4i x[4][QC], qf[4][1][QC];
    paged_k<QC>(g, B, 0, lane, x);
    const uint32_t mul = B.scale(g, g.pages.k_scale, T.h) * (uint32_t)g.score_m;
    const PagedRule<HI> rule(g);
    int lim[4];
    int64_t v[4];  // the largest score; then the row's constant
    uint64_t sum[4];
    const int ranges = (T.keys + pl.span - 1) / pl.span;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int r = 16 * u + ql, near = r < T.live ? r : T.live - 1;
        paged_q<16, QC>(g, pl, T, 16 * u, lane, qf[u]);
        const int sees = T.before + pl.by_group.of(T.row0 + near) + 1;
        lim[u] = sees < k1 ? sees : k1;
        v[u] = INT64_MIN;
        sum[u] = 0;
        if constexpr (PHASE == 2) {
            for (int i = 0; i < ranges; i++) {
                const int64_t y = S.mx[(T.slot + i) * 64 + near];
                v[u] = y > v[u] ? y : v[u];
            }
            v[u] = rule.constant(v[u] == INT64_MIN ? 0 : v[u]);
        }
    }
    const uint32_t last = (uint32_t)g.exp_len - 1;
    if constexpr (PHASE == 2) table_there();
    for (int j = 0; B.key_of(j) < k1; j++) {
        const int key = B.key_of(j);
        const bool pages = ((B.there >> (4 * j)) & 15) == 15;
        v4i next[4][QC];
        paged_k<QC>(g, B, j + 1 < 16 ? j + 1 : 15, lane, next);  // (past the range: no access)
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (u >= tiles) break;
            __builtin_amdgcn_sched_barrier(0);
            v4i D[4];
            paged_dots<16, QC>(x, qf[u], D);
            const int whole = T.before + pl.by_group.of(T.row0 + 16 * u) + 1;
            const bool all = pages && key + 64 <= (whole < k1 ? whole : k1);  // uniform
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int m = paged_of<16>(mul, j, t, lane), k = all ? 4 : B.has(j, t) ? lim[u] - (key + 16 * t + 4 * qg) : 0;
                v4i y = D[t];
                if constexpr (PHASE == 1) {
                    if (!all) {
#pragma unroll
                        for (int e = 1; e < 4; e++) y[e] = e < k ? y[e] : y[0];
                    }
                    const int32_t a = y[0] > y[1] ? y[0] : y[1], b = y[2] > y[3] ? y[2] : y[3];
                    const int64_t z = rule.score(a > b ? a : b, m);
                    if (all || k > 0) v[u] = z > v[u] ? z : v[u];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = (int32_t)rule.index(y[e], m, v[u], last);
                    if (g.table_lds) {
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = s_exp[y[e]];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = g.exp_table[y[e]];
                    }
                    if (!all) {
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = e < k ? y[e] : 0;
                    }
                    sum[u] += (uint64_t)((uint32_t)y[0] + (uint32_t)y[1]) + ((uint32_t)y[2] + (uint32_t)y[3]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < QC; c++) x[t][c] = next[t][c];
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
        if constexpr (PHASE == 1) {
#pragma unroll
            for (int o = 16; o < 64; o <<= 1) {
                const int64_t y = __shfl_xor(v[u], o, 64);
                v[u] = y > v[u] ? y : v[u];
            }
            if (qg == 0) s_x[w][16 * u + ql] = v[u];
        } else {
#pragma unroll
            for (int o = 16; o < 64; o <<= 1) sum[u] += __shfl_xor(sum[u], o, 64);
            if (qg == 0) s_x[w][16 * u + ql] = (int64_t)sum[u];
        }
    }
    __syncthreads();
    if (tid < 64) {
        int64_t y = s_x[0][tid];
#pragma unroll
        for (int i = 1; i < 4; i++) y = PHASE == 2 ? y + s_x[i][tid] : (s_x[i][tid] > y ? s_x[i][tid] : y);
        if constexpr (PHASE == 1) S.mx[(T.slot + T.range) * 64 + tid] = y;
        else S.sum[(T.slot + T.range) * 64 + tid] = (uint64_t)y;
    }
}

// 64 channels from chunk blockIdx.y on. With one range the outputs themselves.
template <int QC, bool HI>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QC == 1 ? 3 : 2))) void k_paged_walk(PagedArgs g, PagedPlan pl, void *scratch) {
    extern __shared__ __attribute__((aligned(1024))) int8_t s_mem[];  // 4 KiB of V a wave, the table
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4, hd = g.pages.hd, c = blockIdx.y;
    int8_t *s_v = s_mem + 4096 * w;
    int32_t *s_exp = (int32_t *)(s_mem + 16384);
    PagedTile T(g, pl, blockIdx.x);
    if (!T.there) return;
    if (g.table_lds) paged_table(g, s_exp, w, 4, lane);
    const int k0 = T.range * pl.span;
    T.rows(g, pl, g.ctx[T.s], g.rows ? g.rows[T.s] : (uint32_t)g.t);
    if (T.live <= 0 || (k0 >= T.keys && T.range > 0)) return;  // the join reads no result of this range
    const int gk1 = k0 + pl.span < T.keys ? k0 + pl.span : T.keys;
    const PagedScratch S = paged_scratch(scratch, pl, hd);
    const int r = 16 * w + ql, near = r < T.live ? r : T.live - 1;
    // the tile's last row sees no more than this
    const int end = 16 * w + 15 < T.live ? 16 * w + 15 : T.live - 1, sees_end = T.before + pl.by_group.of(T.row0 + end) + 1;
    const int k1 = 16 * w >= T.live ? k0 : (sees_end < gk1 ? sees_end : gk1);
    const int sees = T.before + pl.by_group.of(T.row0 + near) + 1, lim = sees < k1 ? sees : k1;
    const int whole0 = T.before + pl.by_group.of(T.row0 + 16 * w) + 1, whole = whole0 < k1 ? whole0 : k1;
    const PagedRule<HI> rule(g);
    const int ranges = (T.keys + pl.span - 1) / pl.span;
    int64_t M = INT64_MIN;
    uint64_t sum = 0;
    for (int i = 0; i < ranges; i++) {
        const int64_t y = S.mx[(T.slot + i) * 64 + near];
        M = y > M ? y : M;
        sum += S.sum[(T.slot + i) * 64 + near];
    }
    const int64_t c0 = rule.constant(M == INT64_MIN ? 0 : M);
    const PagedWeight wt(sum, g.softmax_p, r < T.live);
    const uint32_t last = (uint32_t)g.exp_len - 1;
    v4i qf[1][QC], acc[4][4];
    paged_q<16, QC>(g, pl, T, 16 * w, lane, qf);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[k][i] = v4i{0, 0, 0, 0};
    table_there();
    for (int b0 = k0; b0 < k1; b0 += 1024) {  // 16 blocks with one look at the pages
        PagedBlocks B(g, pl, T.s, b0, 64, 16, lane);
        const int e1 = b0 + 1024 < k1 ? b0 + 1024 : k1;
        B.until(g, pl, T.h, e1, lane);
        v4i x[4][QC], y[4];
        paged_k<QC>(g, B, 0, lane, x);
        const uint32_t mul = B.scale(g, g.pages.k_scale, T.h) * (uint32_t)g.score_m, vs = B.scale(g, g.pages.v_scale, T.h);
        paged_v(g, B, 0, c, lane, y);
        for (int j = 0; B.key_of(j) < e1; j++) {
            v4i D[4];
            paged_dots<16, QC>(x, qf, D);
            __builtin_amdgcn_sched_barrier(0);
            if (j + 1 < 16) paged_k<QC>(g, B, j + 1, lane, x);  // (past the range: no access)
            const int key = B.key_of(j);
            const bool all = ((B.there >> (4 * j)) & 15) == 15 && key + 64 <= whole;  // uniform
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int m = paged_of<16>(mul, j, t, lane);
#pragma unroll
                for (int e = 0; e < 4; e++) D[t][e] = (int32_t)rule.index(D[t][e], m, c0, last);
                if (g.table_lds) {
#pragma unroll
                    for (int e = 0; e < 4; e++) D[t][e] = s_exp[D[t][e]];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) D[t][e] = g.exp_table[D[t][e]];
                }
            }
            if (!all) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const int k = B.has(j, t) ? lim - (key + 16 * t + 4 * qg) : 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) D[t][e] = e < k ? D[t][e] : 0;
                }
            }
            paged_digits<16>(wt, vs, j, lane, s_v, D);
            paged_pv<16>(y, D, lane, s_v, acc, [&] {
                __builtin_amdgcn_sched_barrier(0);
                if (j + 1 < 16) paged_v(g, B, j + 1, c, lane, y);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }
    if (r >= T.live) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int ch = 64 * c + 16 * i + 4 * qg;
        if (ch >= hd) continue;
        int64_t z[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            z[e] = (int64_t)acc[0][i][e] + (int64_t)acc[1][i][e] * 256 + (int64_t)acc[2][i][e] * 65536 + (int64_t)acc[3][i][e] * 16777216;
        if (pl.ng == 1) {
            paged_put(g, pl, T.s, T.h, T.row0 + r, ch, z);
        } else {
            int64_t *to = S.part + ((T.slot + T.range) * 64 + r) * hd + ch;
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = z[e];
        }
    }
}

// The scores of a row over PG_CHUNK keys to their entries, in place, and the entries' sum.
template <bool HI>
__global__ __launch_bounds__(256) void k_paged_entries(PagedArgs g, PagedPlan pl, void *scratch) {
    typedef typename std::conditional<HI, int32_t, int64_t>::type Score;
    constexpr Score LOW = HI ? (Score)INT32_MIN : (Score)INT64_MIN;
    constexpr int N = PG_CHUNK / 256;
    extern __shared__ __attribute__((aligned(1024))) int32_t s_exp[];  // the table, where it fits
    __shared__ uint64_t s_sum[4];
    const PagePool &p = g.pages;
    const int tid = threadIdx.x;
    if (g.table_lds) paged_table(g, s_exp, tid >> 6, 4, tid & 63);
    // (row fastest, then the chunk)
    const int r = blockIdx.x % pl.rows, chunk = blockIdx.x / pl.rows % pl.chunks;
    PagedTile T;
    T.place = blockIdx.x / pl.rows / pl.chunks;
    T.panel = pl.by_tiles.of((int)T.place);
    T.tile = (int)T.place - T.panel * pl.tiles;
    T.s = pl.by_heads.of(T.panel);
    T.rows(g, pl, g.ctx[T.s], g.rows ? g.rows[T.s] : (uint32_t)g.t);
    if (r >= T.live) return;
    const size_t place = T.place;
    const int keys = T.keys;  // of the tile: those have scores, in whole blocks
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
        y[i] = (int32_t)(d < last ? d : last);
    }
    table_there();
    if (g.table_lds) {
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = s_exp[y[i]];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = g.exp_table[y[i]];
    }
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = x[i] == LOW ? 0 : y[i];
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
    const int hd = g.pages.hd, quads = hd / 4;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, at = i / quads;  // (tile of a panel, row)
    const int ch = 4 * (int)(i - at * quads);
    PagedTile T;
    T.place = at / pl.rows;
    const int r = (int)(at - T.place * pl.rows);
    if (T.place >= (size_t)pl.panels * pl.tiles) return;
    T.panel = pl.by_tiles.of((int)T.place);
    T.tile = (int)T.place - T.panel * pl.tiles;
    T.s = pl.by_heads.of(T.panel);
    T.h = T.panel - T.s * g.pages.kv_heads;
    T.rows(g, pl, g.ctx[T.s], g.rows ? g.rows[T.s] : (uint32_t)g.t);
    if (r >= T.live) return;
    const int ranges = T.keys > pl.span ? (T.keys + pl.span - 1) / pl.span : 1;
    const PagedScratch S = paged_scratch(scratch, pl, hd);
    int64_t x[4] = {0, 0, 0, 0};
    const int64_t *from = S.part + (T.place * pl.ng * pl.rt + r) * hd + ch;
    for (int c0 = 0; c0 < ranges; c0 += 8) {  // eight in flight
        int64_t y[8][4];
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) y[c][e] = from[(size_t)(c0 + c < ranges ? c0 + c : c0) * pl.rt * hd + e];
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] += c0 + c < ranges ? y[c][e] : 0;
    }
    paged_put(g, pl, T.s, T.h, T.row0 + r, ch, x);
}

static PagedPlan paged_plan(const PagedArgs &g) {
    PagedPlan p;
    p.group = g.heads / g.pages.kv_heads;
    const long long rows = (long long)g.t * p.group;
    p.panels = g.streams * g.pages.kv_heads;
    // Keys of a tile in one launch, whose dots fit the registers of its waves. It reads K and V and nothing else; several launches
    // write and read the scores too, but spread a panel over the chip. In us, one launch and several, with three quarters of the
    // keys there in the mean: 768 panels of 8,192 keys 117 and 155, 12 panels 27 and 36; of 16,000 keys 768 panels 238 and 290, 200 panels 71 and 89, 156 panels 66 and 77, 132 panels
    // 62 and 67, 120 panels 60 and 59, 96 panels 59 and 50, 48 panels 50 and 34 (of 9,000 keys the sides meet at some 80 panels).
    // 16 rows (8 query heads of 128 channels, 128 panels of 2,000 keys) 25 and 38.
    const int most = rows > 8 || (rows > 4 && g.pages.hd > 128) ? 2048 : rows > 4 ? 4096 : g.pages.hd > 128 ? 4096 : g.pages.hd > 64 || p.panels < 128 ? 8192 : 16384;
    // 64 rows: 16 streams of 64 rows over 4,096 keys 100 us, in tiles of 16 rows 155. 4 rows: a row of 1,000 keys 9.2 us, as one
    // of 16 rows 12.2 (768 panels 20.5 and 23.8).
    p.rt = rows <= 4 ? 4 : rows <= 8 && g.keys <= most ? 8 : rows <= 16 || g.keys <= most ? 16 : 64;
    p.rows = rows < p.rt ? (int)rows : p.rt;
    p.tiles = (int)((rows + p.rt - 1) / p.rt);
    while (1 << p.page_log < g.pages.page) p.page_log++;
    p.span = (g.keys + 63) / 64 * 64;
    if (g.keys > most) {
        const long long wgs = (long long)p.panels * p.tiles;
        auto ranges = [&](int least_keys, long long all) {
            long long ng = (all + wgs - 1) / wgs;
            const long long least = (g.keys + 4095) / 4096, more = (g.keys + least_keys - 1) / least_keys;
            ng = ng < least ? least : (ng > more ? more : ng);
            p.span = (int)(((g.keys + ng - 1) / ng + 255) / 256) * 256;
            p.ng = (g.keys + p.span - 1) / p.span;
        };
        // workgroups for each of 256 CUs, in us of whole calls (three quarters of the keys there in the mean):
        //                                                        1      2      3      4      8     12     16
        //   one row, 200 panels of up to 32,000 keys                  170    171    171    164    164    161
        //   one row, 100 panels, 16,000                              58.8   59.2   59.9   57.9   58.1   58.3
        //   one row, 128 panels of 128 channels, 12,000              85.5   87.5   85.2   84.7   84.6   85.1
        //   eight rows, 128 panels of 128 channels, 6,000     68.7   67.8   74.0   71.9   76.3
        //   16 rows, 128 panels, 4,000                        49.9   47.4   49.6   51.3   51.0
        //   12 rows, 48 panels, 8,000                         42.4   39.7   40.7   41.0   41.0
        //   64 rows, 192 panels, 4,096                         113    103          99.5    112
        //   256 rows, 48 panels, 8,000                         195    151           144    161
        //   256 rows, 12 panels, 16,000                        148    126           156    194
        // (one stream's 256 rows alone would have two)
        if (p.rt == 4) ranges(1024, 12 * 256);
        else if (p.rt == 16) ranges(512, 2 * 256);
        else ranges(512, 4 * 256);
        p.store = p.rt < 64;
        p.split = 1;
        p.chunks = p.store ? (g.keys + PG_CHUNK - 1) / PG_CHUNK : p.ng;
    }
    p.by_group = PagedDiv((uint32_t)p.group);
    p.by_tiles = PagedDiv((uint32_t)p.tiles);
    p.by_heads = PagedDiv((uint32_t)g.pages.kv_heads);
    p.by_inner = PagedDiv((uint32_t)(8ll * p.tiles * p.ng));
    return p;
}

// A grid has fewer than 2^32 threads: workgroups of up to 1,024 in one launch, and 256 in each of several.
bool paged_fits(const PagedArgs &g) {
    const PagedPlan p = paged_plan(g);
    const long long tiles = (long long)p.panels * p.tiles;
    return ((long long)p.panels + 7) * p.tiles < (1ll << 22) / p.ng && (!p.store || tiles * p.rows < (1ll << 23) / p.chunks) &&
           tiles * p.rt < (1ll << 31) / (g.pages.hd / 4);
}

size_t paged_workspace(const PagedArgs &g) {
    const PagedPlan p = paged_plan(g);
    size_t bytes = 0;
    if (p.split) paged_scratch(nullptr, p, g.pages.hd, &bytes);
    return bytes;
}

template <int RT, int QC, int NB, int NW, bool HI>
static hipError_t launch_paged_t(const PagedArgs &g, const PagedPlan &p, hipStream_t stream) {
    const int acc = (8 * QC * RT * PG_ACC + 1023) / 1024 * 1024;
    const int table = RT >= 8 && g.table_lds ? 1024 * ((g.exp_len + 255) / 256) : 0;
    const size_t lds = (size_t)(table > acc ? table : acc) + 4096 * NW + 16 * NW * RT;
    const hipError_t e = allow_dynamic_lds((const void *)k_paged_tile<RT, QC, NB, NW, HI>, lds);
    if (e != hipSuccess) return e;
    launch_k((k_paged_tile<RT, QC, NB, NW, HI>), dim3((unsigned)((p.panels + 7) / 8 * 8) * p.tiles * p.ng), dim3(64 * NW), lds, stream, g, p);
    return hipGetLastError();
}

template <int RT, int QC, bool HI>
static hipError_t launch_paged_q(const PagedArgs &g, const PagedPlan &p, void *scratch, hipStream_t stream) {
    if constexpr (RT != 8) if (p.split) {
        hipError_t e;
        const unsigned grid = (unsigned)((p.panels + 7) / 8 * 8) * p.tiles * p.ng;
        const size_t table = g.table_lds ? (size_t)1024 * ((g.exp_len + 255) / 256) : 0;
        auto run = [&](auto kernel, dim3 n, size_t lds) {
            const hipError_t f = allow_dynamic_lds((const void *)kernel, lds);
            if (f != hipSuccess) return f;
            launch_k(kernel, n, dim3(256), lds, stream, g, p, scratch);
            return hipGetLastError();
        };
        if (p.store) {
            constexpr int GC = QC == 4 ? 2 : QC;  // (the sums of more channels do not fit the registers)
            if ((e = run(k_paged_scores<RT, QC, HI>, dim3(grid), 0)) != hipSuccess) return e;
            if ((e = run(k_paged_entries<HI>, dim3((unsigned)p.panels * p.tiles * p.chunks * p.rows), table)) != hipSuccess) return e;
            if ((e = run(k_paged_products<RT, GC, HI>, dim3(grid, QC / GC), 0)) != hipSuccess) return e;
        } else if constexpr (RT == 16) {
            if ((e = run(k_paged_scan<QC, HI, 1>, dim3(grid), 0)) != hipSuccess) return e;
            if ((e = run(k_paged_scan<QC, HI, 2>, dim3(grid), table)) != hipSuccess) return e;
            if ((e = run(k_paged_walk<QC, HI>, dim3(grid, (g.pages.hd + 63) / 64), 16384 + table)) != hipSuccess) return e;
            if (p.ng == 1) return hipSuccess;
        }
        const size_t quads = (size_t)p.panels * p.tiles * p.rows * (g.pages.hd / 4);
        return run(k_paged_out, dim3((unsigned)((quads + 255) / 256)), 0);
    }
    // Blocks a wave and waves, by the keys a call may read (three quarters of them there in the mean of these figures). One row a panel: a workgroup a CU and less takes 16 waves, whose
    // chains are short (12 panels of 1,000 keys 8.6 us, in four waves 9.3); 768 panels one round of three workgroups a CU (18.9
    // us at 1,024 keys); more keys two workgroups of eight waves a CU, one at its loads while the other works (2,048 keys
    // 37.9 us, in one of 16 waves 46.0; 4,096 keys 62.8 and 70.2, and with 128 channels 166 and 141, where eight blocks spill).
    if (p.span <= 256) return launch_paged_t<RT, QC, 1, 4, HI>(g, p, stream);
    if (p.span <= 1024) {
        if constexpr (RT <= 8)
            if (p.panels <= 256) return launch_paged_t<RT, QC, 1, 16, HI>(g, p, stream);
        return launch_paged_t<RT, QC, 4, 4, HI>(g, p, stream);
    }
    if (p.span <= 2048) return launch_paged_t<RT, QC, 4, 8, HI>(g, p, stream);
    if constexpr (RT == 8 && QC <= 2) return launch_paged_t<RT, QC, 4, 16, HI>(g, p, stream);
    if constexpr (RT == 4) {
        if (p.span <= 4096) return launch_paged_t<RT, QC, QC == 2 ? 4 : 8, QC == 2 ? 16 : 8, HI>(g, p, stream);
        if constexpr (QC <= 2)
            if (p.span <= 8192) return launch_paged_t<RT, QC, 8, 16, HI>(g, p, stream);
        if constexpr (QC == 1) return launch_paged_t<RT, QC, 16, 16, HI>(g, p, stream);
    }
    return hipErrorInvalidValue;  // (the plan splits longer ones)
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
    return p.rt == 4 ? launch_paged_r<4>(g, p, workspace, stream) : p.rt == 8 ? launch_paged_r<8>(g, p, workspace, stream) : launch_paged_r<16>(g, p, workspace, stream);
}

}  // namespace hs
