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
// the keys as in k_attend (the row max, the sum of the entries, p and sum p v). It is for what the other forms
// do not take, not for speed: each row walks K and V again, and a key's weight goes through a lane move to all lanes. 768
// panels of 16 rows at 500 to 1,000 keys: head_dim 20 625 us, 60 927 (64 in tiles 21.6); 12 panels of 8 rows at 100 keys 25.
__global__ __launch_bounds__(256) void k_rows(RowsArgs g, int s0, int n_tasks) {
    __shared__ __attribute__((aligned(16))) int s_q[4][64];
    const AttnArgs &a = g.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int task = blockIdx.x * 4 + wave;
    const int row = task < n_tasks ? task / a.n_head : 0, h = task < n_tasks ? task % a.n_head : 0;
    const int at = row / g.t, i = row - at * g.t, s = s0 + at, hd = a.hd;  // (s0: the launch's first stream)
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

// ---- Tiles of 16 rows on MFMA ------------------------------------------------------------------------
// One workgroup of NW waves takes 16 rows of one (stream, head); wave w the key blocks (64 keys) w, w + NW, ..,
// at most NB of them, so every dot of the tile stays in registers (NB x 16 a lane) from the one product with K to
// the product with V: K and V are read once. K is the first operand of v_mfma_i32_16x16x64_i8, so lane l holds
// the dots of row l % 16 with keys 16 t + 4 (l / 16) + e of a block. The steps are those of k_attend_short: the
// extreme dots (the score is monotone in the dot), the table entries and their sum, p as four balanced i8
// digits, four products with V^T by transposing LDS reads; here the waves share the keys of the same rows, so the
// extremes and the sums meet in LDS, and the output sums in 64-bit LDS atomics (integers: any order).
// QC: 64-byte chunks of a head (the last one may be part empty: its lanes hold zeros).
// 768 panels of 16 rows at 750 keys (76 MB): 21.6 us, 3.5 TB/s; 12 panels 6.4 us at 100 keys. Few panels are bound by
// the chain of one workgroup (loads, two exchanges between the waves, products), many by HBM and, from three tiles a
// panel on, by VALU issue. Counted at 512 and 1,024 keys: a block takes 272 VALU instructions, 17 a score; a wave's
// fixed part 380 (320 where it has no block), which eight waves a tile pay for one or two blocks each. Causal chunks of up
// to 256 rows, 192 panels: 52 us, of them 27 of VALU issue: 16.9 M instructions, 7.4 M for 27,200 blocks and the rest,
// some 480 a wave with the masks, fixed. More rows a workgroup would share that part; it is not tried.
// 65 to 128 channels: 128 panels of 23 rows at 1,500 keys (50 MB) 23.3 us; 129 to 256: 128 panels of 16 rows at 750 keys (51 MB)
// 21.4. There the loads of a channel group leave only under the products of the one before.
constexpr int RT_ROWS = 16;
constexpr int RT_TABLE = 16384;  // entries of the table copied to LDS at most
constexpr int RT_ACC = 66;       // 64 channels' sums of a row and two of padding (bank spread)

// Sums over the 16 rows (lanes l % 16) of p of a block's 64 keys, given as p + 0x80808080: lane l receives the sum of
// key 16 (l % 16 / 4) + 4 (l / 16) + l % 4. A reduce-scatter in four steps: each lane hands half of what it holds
// to its partner and keeps the other half.
__device__ __forceinline__ uint64_t row_sums(const uint32_t (&p)[16], int lane) {
    const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2, b0 = lane & 1;
    uint32_t x[8];  // two rows: at most 2^31
#pragma unroll
    for (int i = 0; i < 8; i++)
        x[i] = (b3 ? p[i + 8] : p[i]) + (uint32_t)dpp_mov<0x140>((int32_t)(b3 ? p[i] : p[i + 8])) - 0x01010100u;
    uint64_t y[4], z[2];
#pragma unroll
    for (int i = 0; i < 4; i++)
        y[i] = (uint64_t)(b2 ? x[i + 4] : x[i]) + (uint32_t)dpp_mov<0x141>((int32_t)(b2 ? x[i] : x[i + 4]));
#pragma unroll
    for (int i = 0; i < 2; i++) z[i] = (b1 ? y[i + 2] : y[i]) + (uint64_t)lane_move64<1>((int64_t)(b1 ? y[i] : y[i + 2]));
    return (b0 ? z[1] : z[0]) + (uint64_t)lane_move64<0>((int64_t)(b0 ? z[0] : z[1]));
}

// What a lane needs to know of its row (l % 16): which keys it sees.
struct RowSight {
    int base, lim;   // keys up to lim are seen: the context (tree), the row's own key (causal)
    int count;       // nodes of the stream (tree; else 0)
    uint64_t word;   // tree: word l / 16 of the row's mask
};

__device__ __forceinline__ RowSight row_sight(const RowsArgs &g, const StreamRows &R, int row, int qg, int keys) {
    RowSight v;
    const bool live = row < R.count;
    v.base = R.base;
    v.lim = live ? (g.mask ? (R.base < keys ? R.base : keys) - 1 : (R.base + row < keys - 1 ? R.base + row : keys - 1)) : -1;
    v.count = g.mask ? R.count : 0;
    v.word = g.mask && live && qg < g.words ? R.mask[(size_t)row * g.words + qg] : 0;
    return v;
}

// Of the keys 64 kb + 16 t + 4 (l / 16) + e those that the row sees, bit 4 t + e. (Every lane of the wave.)
__device__ __forceinline__ uint32_t sight_bits(const RowSight &v, int kb, int lane, int keys) {
    const int seen = v.lim + 1 - 64 * kb;
    uint64_t m = seen >= 64 ? ~(uint64_t)0 : (seen > 0 ? ((uint64_t)1 << seen) - 1 : 0);
    const int n0 = 64 * kb - v.base;  // the node of the first key
    if (v.count && n0 + 63 >= 0) {    // uniform
        // the 64 mask bits from node n0 on, those of nodes count .. and of keys past the cache cleared
        const int words = (v.count + 63) >> 6, w = n0 >> 6, o = n0 & 63;
        const uint64_t lo = __shfl(v.word, 16 * (w & 3) + (lane & 15), 64), hi = __shfl(v.word, 16 * ((w + 1) & 3) + (lane & 15), 64);
        uint64_t n = w >= 0 && w < words ? lo >> o : 0;
        if (o && w + 1 < words) n |= hi << (64 - o);
        const int most = (v.count < keys - v.base ? v.count : keys - v.base) - n0;  // nodes up to the end of the block
        n = most <= 0 ? 0 : (most < 64 ? n & (((uint64_t)1 << most) - 1) : n);
        m |= n0 < 0 ? n & ~(uint64_t)0 << -n0 : n;
    }
    m >>= 4 * (lane >> 4);
    return (uint32_t)(m & 15) | (uint32_t)(m >> 12 & 0xf0) | (uint32_t)(m >> 24 & 0xf00) | (uint32_t)(m >> 36 & 0xf000);
}

// ---- The steps on a block: 64 keys x 16 rows, D[t][e] of lane l belongs to row l % 16 and key 16 t + 4 (l / 16) + e

// The largest and smallest dot among the keys the row sees.
__device__ __forceinline__ void block_extremes(const v4i (&D)[4], bool all, uint32_t ok, int32_t &dmax, int32_t &dmin) {
    if (all) {  // uniform
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                dmax = D[t][e] > dmax ? D[t][e] : dmax;
                dmin = D[t][e] < dmin ? D[t][e] : dmin;
            }
    } else {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool in = (ok >> (4 * t + e)) & 1;
                const int32_t hi = in ? D[t][e] : INT32_MIN, lo = in ? D[t][e] : INT32_MAX;
                dmax = hi > dmax ? hi : dmax;
                dmin = lo < dmin ? lo : dmin;
            }
    }
}

// The table index min(M - score(dot), last) of a row whose extreme dots are dmax and dmin (the score is monotone
// in the dot, so M is the score of one of them). Shifts from 32 to 60 (HI; m > -2^31): with x = the high word of
// dot m + 2^(s-1) and h = s - 32 the score is x >> h, |x| <= 2^21 + 2^27, and
//   M - (x >> h) = (M 2^h + 2^h - 1 - x) >> h,  -x = the high word of -dot m + 2^32 - 1 - 2^(s-1),
// so one multiply-add with the row's constant, a shift and a minimum give the index (a masked key's may be
// negative: as an unsigned number it is past the table, and its entry is not used).
template <bool HI>
struct RowIndex {
    int64_t c;  // HI: the row's addend; else M
    __device__ __forceinline__ explicit RowIndex(int64_t row) : c(row) {}
    __device__ __forceinline__ RowIndex(const AttnArgs &a, int32_t dmax, int32_t dmin) {
        if (dmax < dmin) dmax = dmin = 0;  // a row that sees nothing
        const int64_t s0 = attn_score<HI>(a, dmax), s1 = attn_score<HI>(a, dmin);
        const int64_t M = s0 > s1 ? s0 : s1;
        const int h = a.score_s - 32;
        if constexpr (HI) c = (((M + 1) << h) - 1) * ((int64_t)1 << 32) + 0xffffffffll - ((int64_t)1 << (a.score_s - 1));
        else c = M;
    }
    __device__ __forceinline__ int32_t at(const AttnArgs &a, int32_t dot, int32_t last) const {
        if constexpr (HI) {
            const int64_t y = (int64_t)dot * (-a.score_m) + c;
            const uint32_t i = (uint32_t)((int32_t)(y >> 32) >> (a.score_s - 32));
            return (int32_t)(i < (uint32_t)last ? i : (uint32_t)last);
        } else {
            return (int32_t)clamp64(c - attn_score<false>(a, dot), 0, last);
        }
    }
};

// The dots of a block to its table entries, in place (0 where the row does not see the key).
template <bool HI>
__device__ __forceinline__ void block_entries(const AttnArgs &a, v4i (&D)[4], const RowIndex<HI> &ix, const int32_t *s_exp,
                                              int32_t last, bool all, uint32_t ok) {
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) D[t][e] = ix.at(a, D[t][e], last);
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) D[t][e] = s_exp[D[t][e]];
    if (!all) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) D[t][e] = (ok >> (4 * t + e)) & 1 ? D[t][e] : 0;
    }
}

// Their sum (entries are below 2^31: a pair sums in 32 bits).
__device__ __forceinline__ uint64_t block_sum(const v4i (&D)[4]) {
    uint64_t s = 0;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e += 2) s += (uint32_t)D[t][e] + (uint32_t)D[t][e + 1];
    return s;
}

// The entries of a block to the digit planes of p = floor(e 2^P / S), in place: D[k] word t holds digit k of keys
// 16 t + 4 (l / 16) + e. The rule of softmax_p_of with 0x80808080 inside the rounding constant: the low word of the sum
// is p + 0x80808080 at once, whose bytes xor 0x80 are the balanced digits. Where `mass` is set, each key's weights
// summed over the 16 rows are added to it.
__device__ __forceinline__ void block_digits(v4i (&D)[4], double R, double sp, uint64_t *mass, int keys, int lane) {
    constexpr double magic = 6755399441055744.0 + 2155905152.0;  // 1.5 2^52 + 0x80808080
    uint32_t o[4][4], dg[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const double ed = (double)(uint32_t)D[i >> 2][i & 3], w = fma(ed, R, magic), r = fma(w - magic, sp, ed);
        dg[i] = (uint32_t)__double2loint(w) + (uint32_t)(__double2hiint(r) >> 31);
    }
    if (mass) {  // uniform
        const uint64_t x = row_sums(dg, lane);
        const int key = 16 * ((lane & 15) >> 2) + 4 * (lane >> 4) + (lane & 3);
        if (x && key < keys) atomicAdd((unsigned long long *)mass + key, (unsigned long long)x);
    }
#pragma unroll
    for (int t = 0; t < 4; t++) byte_transpose(dg[4 * t], dg[4 * t + 1], dg[4 * t + 2], dg[4 * t + 3], o[t]);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int t = 0; t < 4; t++) D[k][t] = (int32_t)(o[t][k] ^ 0x80808080u);
}

// The factors of p of a row (softmax_p_of); rows that are not there and rows without weight: p = 0 (R = 0).
struct RowWeight {
    double R, sp;
    __device__ __forceinline__ RowWeight(uint64_t sum, int P, bool live)
        : R(sum > 0 && live ? ldexp(1.0 / (double)sum, P) : 0.0), sp(softmax_sp(sum, P)) {}
};

// acc[k][i] += V^T digits over a block whose V rows lie in s_v (16-byte chunk c of row r at slot 4 r + (c ^ vsw(r))):
// channel 16 i + 4 (l / 16) + e of row l % 16.
__device__ __forceinline__ void block_pv(const int8_t *s_v, const v4i (&pf)[4], int lane, v4i (&acc)[4][4]) {
    const int ql = lane & 15, qg = lane >> 4, tr_k = ql >> 1, key0 = 16 * (tr_k >> 2) + 4 * qg + (tr_k & 3);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int8_t *p0 = s_v + (4 * key0 + (i ^ vsw<4>(key0 & 15))) * 16 + 8 * (ql & 1);
        const v2i r0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)p0);
        const v2i r1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(p0 + 32 * 64));
        const v4i vf = v4i{r0[0], r0[1], r1[0], r1[1]};
#pragma unroll
        for (int k = 0; k < 4; k++) acc[k][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf, pf[k], acc[k][i], 0, 0, 0);
    }
}

__device__ __forceinline__ int64_t plane_sum(const v4i (&acc)[4][4], int i, int e) {
    return (int64_t)acc[0][i][e] + (int64_t)acc[1][i][e] * 256 + (int64_t)acc[2][i][e] * 65536 +
           (int64_t)acc[3][i][e] * 16777216;
}

// The rows of a (stream, head) in a cache, read by buffer loads: one offset a lane for all blocks and the block's in
// a scalar register; rows past the cache read as zeros without an access, and so does all of a block without keys
// (`none`), so nothing is clamped. K comes as the product's operand (chunk c: 16 bytes from 64 c + 16 (l / 16) on of
// rows 16 t + l % 16), V in block_pv's layout (group c: the 16 bytes (l % 4) ^ vsw of rows 16 u + l / 4). Columns
// past the head read its first ones: K's meet zeros of q there, V's outputs are not stored.
struct Panel {
    __amdgpu_buffer_rsrc_t rsrc;
    int bytes;  // at most 2^30
    __device__ __forceinline__ Panel(const int8_t *p, int cap, int hd) : bytes(cap * hd) {
        rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, bytes, 0x00020000);
    }
    // the 16 bytes at lane offset `at` of the block that starts at row `row` (below cap), or zeros
    __device__ __forceinline__ v4i load(int at, int row, int hd, bool none) const {
        return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, none ? bytes : row * hd, 0));
    }
};
template <int QC>
__device__ __forceinline__ void load_k(const Panel &p, int row, int c, int hd, bool none, int lane, v4i (&x)[4][QC]) {
    const int o = 64 * c + 16 * (lane >> 4), at = (lane & 15) * hd + (o < hd ? o : 0);
#pragma unroll
    for (int t = 0; t < 4; t++) x[t][c] = p.load(at + 16 * t * hd, row, hd, none);
}
__device__ __forceinline__ void load_v(const Panel &p, int row, int c, int hd, bool none, int lane, v4i (&x)[4]) {
    const int r = lane >> 2, o = 64 * c + 16 * ((lane & 3) ^ vsw<4>(r)), at = r * hd + (o < hd ? o : 0);
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = p.load(at + 16 * u * hd, row, hd, none);
}

// The table to LDS: whole KiB straight, the end entry by entry (places past it repeat the last one). The caller waits.
__device__ __forceinline__ void load_table(const AttnArgs &a, int32_t *s_exp, int w, int waves, int lane) {
    const int whole = a.exp_len / 256;
    for (int ch = w; ch < whole; ch += waves)
        __builtin_amdgcn_global_load_lds((const void *)(a.exp_table + ch * 256 + 4 * lane), (lds_void *)(s_exp + ch * 256), 16, 0, 0);
    if (w == 0)
        for (int i = 256 * whole + lane; i < (a.exp_len + 255) / 256 * 256; i += 64)
            s_exp[i] = a.exp_table[i < a.exp_len ? i : a.exp_len - 1];
}

// The bytes of LDS before a tile's V regions: the table, which the sums of the outputs take over.
__host__ __device__ inline int tile_top(int qc, int table_chunks) {
    const int acc = (8 * qc * RT_ROWS * RT_ACC + 1023) / 1024 * 1024;
    return 1024 * table_chunks > acc ? 1024 * table_chunks : acc;
}

template <int QC, int NB, int NW, bool HI>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void k_rows_tile(RowsArgs g, int tiles, int panels) {
    static_assert(NB <= 4, "the plane sums of a wave's keys in 32 bits");
    extern __shared__ __attribute__((aligned(1024))) int8_t s_mem[];
    const AttnArgs &a = g.a;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4;
    // workgroup L runs on XCD L % 8: the tiles of a panel stay on one XCD and share K and V in its L2
    const int L = blockIdx.x, panel = L / (8 * tiles) * 8 + (L & 7), tile = (L >> 3) % tiles;
    if (panel >= panels) return;
    const int s = panel / a.n_head, h = panel - s * a.n_head, hd = a.hd;
    const StreamRows R = stream_rows(g, s);
    const int row0 = RT_ROWS * tile, row = row0 + ql;
    if (row0 >= R.count) return;
    const int last = a.exp_len - 1, table_chunks = (a.exp_len + 255) / 256;
    int32_t *s_exp = (int32_t *)s_mem;
    const int top = tile_top(QC, table_chunks);
    int64_t *s_acc = (int64_t *)s_mem;  // [QC][16][RT_ACC], over the table when that is done with
    int8_t *s_v = s_mem + top + 4096 * w;
    uint64_t *s_sum = (uint64_t *)(s_mem + top + 4096 * NW);  // [NW][16]
    int32_t *s_mm = (int32_t *)(s_sum + NW * RT_ROWS);        // [2][NW][16]

    int keys = stream_keys(g, R);
    if (!g.mask) keys = R.base + row0 + RT_ROWS < keys ? R.base + row0 + RT_ROWS : keys;  // causal: the tile's last row
    keys = keys < 64 * NB * NW ? keys : 64 * NB * NW;  // (the launch's bound holds every count)
    const size_t at = (size_t)R.slot * a.n_head + h, base = at * a.ctx_cap * hd;
    const Panel K(a.kc + base, a.ctx_cap, hd), V(a.vc + base, a.ctx_cap, hd);
    auto block = [&](int j) { return NW * j + w; };
    auto mine = [&](int j) { return 64 * block(j) < keys; };  // uniform

    const v4i zero = v4i{0, 0, 0, 0};
    load_table(a, s_exp, w, NW, lane);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);  // the table's loads before those of K: who has K has the table
    v4i qf[QC];
#pragma unroll
    for (int c = 0; c < QC; c++) {
        const int o = 64 * c + 16 * qg;
        qf[c] = row < R.count && o < hd ? *(const v4i *)(a.q + (size_t)(R.first + row) * a.ldq + h * hd + o) : zero;
    }

    const RowSight sight = row_sight(g, R, row, qg, keys);
    // K, then V of the first channel group, all in flight together and no branch around them, so that the waits count
    // them exactly; a block's dots take the registers of its K
    v4i D[NB][4], vr[NB][4];
    auto v_load = [&](int j, int c) { load_v(V, 64 * block(j), c, hd, !mine(j), lane, vr[j]); };
    v4i kr[NB][4][QC <= 2 ? QC : 1];
    if constexpr (QC <= 2) {
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int c = 0; c < QC; c++) load_k<QC>(K, 64 * block(j), c, hd, !mine(j), lane, kr[j]);
#pragma unroll
        for (int j = 0; j < NB; j++) v_load(j, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                if (mine(j)) {
                    D[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[j][t][0], qf[0], zero, 0, 0, 0);
                    if (QC == 2) D[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[j][t][QC == 2], qf[QC == 2], D[j][t], 0, 0, 0);
                }
    } else {
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (!mine(j)) continue;
            v4i k4[4][QC];
#pragma unroll
            for (int c = 0; c < QC; c++) load_k<QC>(K, 64 * block(j), c, hd, false, lane, k4);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                D[j][t] = zero;
#pragma unroll
                for (int c = 0; c < QC; c++) D[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k4[t][c], qf[c], D[j][t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int j = 0; j < NB; j++) v_load(j, 0);
    }

    // a block whose keys every row of the tile sees
    const int whole = g.mask ? R.base : R.base + row0 + 1;
    auto all = [&](int j) { return 64 * block(j) + 64 <= (whole < keys ? whole : keys); };
    uint32_t ok[NB];
    int32_t dmax = INT32_MIN, dmin = INT32_MAX;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        ok[j] = 0;
        if (!mine(j)) continue;
        if (!all(j)) ok[j] = sight_bits(sight, block(j), lane, keys);
        block_extremes(D[j], all(j), ok[j], dmax, dmin);
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {  // the four lanes of the row
        const int32_t x = __shfl_xor(dmax, o, 64), y = __shfl_xor(dmin, o, 64);
        dmax = x > dmax ? x : dmax;
        dmin = y < dmin ? y : dmin;
    }
    if (qg == 0) {
        s_mm[w * RT_ROWS + ql] = dmax;
        s_mm[(NW + w) * RT_ROWS + ql] = dmin;
    }
    if (!mine(0)) wait_vmcnt<0>();  // (no K to wait for)
    lds_barrier();                  // not the fence of __syncthreads, which would wait for V too
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const int32_t x = s_mm[i * RT_ROWS + ql], y = s_mm[(NW + i) * RT_ROWS + ql];
        dmax = x > dmax ? x : dmax;
        dmin = y < dmin ? y : dmin;
    }
    const RowIndex<HI> ix(a, dmax, dmin);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (!mine(j)) continue;
        block_entries<HI>(a, D[j], ix, s_exp, last, all(j), ok[j]);
        sum += block_sum(D[j]);
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (qg == 0) s_sum[w * RT_ROWS + ql] = sum;
    lds_barrier();
    sum = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) sum += s_sum[i * RT_ROWS + ql];
    for (int i = tid; i < QC * RT_ROWS * RT_ACC; i += 64 * NW) s_acc[i] = 0;  // (every wave has its entries)
    const RowWeight wt(sum, a.softmax_p, row < R.count);
#pragma unroll
    for (int j = 0; j < NB; j++) {
        __builtin_amdgcn_sched_barrier(0);  // (a block at a time: interleaved they spill)
        if (mine(j))
            block_digits(D[j], wt.R, wt.sp, g.mass ? g.mass + at * a.ctx_cap + 64 * block(j) : nullptr, keys - 64 * block(j), lane);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < QC; c++) {
        v4i acc[4][4];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[k][i] = zero;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (!mine(j)) continue;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 4; u++) *(v4i *)(s_v + 1024 * u + 16 * lane) = vr[j][u];
            if (c + 1 < QC) v_load(j, c + 1);
            block_pv(s_v, D[j], lane, acc);
        }
        if (c == 0) lds_barrier();  // the zeros
        if (mine(0)) {
            unsigned long long *to = (unsigned long long *)s_acc + (c * RT_ROWS + ql) * RT_ACC + 4 * qg;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    // (at most 256 keys a wave: a plane's sum is below 2^22, two planes' below 2^31)
                    const int32_t lo = acc[0][i][e] + acc[1][i][e] * 256, hi = acc[2][i][e] + acc[3][i][e] * 256;
                    atomicAdd(to + 16 * i + e, (unsigned long long)((int64_t)hi * 65536 + lo));
                }
        }
    }
    lds_barrier();
    const double mo = a.out_s > 95 ? 0.0 : ldexp((double)a.out_m, -a.out_s);
    for (int i = tid; i < RT_ROWS * hd / 4; i += 64 * NW) {
        const int r = i / (hd / 4), ch = 4 * (i - r * (hd / 4));
        if (row0 + r >= R.count) break;
        const int64_t *x = s_acc + ((ch >> 6) * RT_ROWS + r) * RT_ACC + (ch & 63);
        uint32_t packed = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) packed |= (uint32_t)(uint8_t)(int8_t)attn_out_byte(x[e], mo, a.out_m, a.out_s) << (8 * e);
        *(uint32_t *)attn_out(a, R.first + row0 + r, h * hd + ch) = packed;
    }
}

template <int QC, int NB, int NW, bool HI>
static hipError_t launch_tile_t(const RowsArgs &g, hipStream_t stream) {
    const int tiles = (g.t + RT_ROWS - 1) / RT_ROWS, panels = g.streams * g.a.n_head;
    const size_t lds = (size_t)tile_top(QC, (g.a.exp_len + 255) / 256) + 4096 * NW + 16 * NW * RT_ROWS;
    const hipError_t e = allow_dynamic_lds((const void *)k_rows_tile<QC, NB, NW, HI>, lds);
    if (e != hipSuccess) return e;
    launch_k((k_rows_tile<QC, NB, NW, HI>), dim3((unsigned)((panels + 7) / 8 * 8) * tiles), dim3(64 * NW), lds, stream, g, tiles, panels);
    return hipGetLastError();
}

// Waves and blocks a wave by the keys the caches hold. Up to 1,024 keys eight waves of two blocks: against four of four,
// one stream of 12 heads and 16 rows at 700 keys 9.3 us and 11.9, 64 streams 21.2 and 23.5, 128 streams 39.0 and 40.2.
// Above 64 channels that holds while there is a workgroup a CU at most (12 panels at head_dim 128: 13.3 us and 14.9;
// 768: 46.6 and 42.3: of the eight waves' form only one workgroup fits a CU).
template <int QC, bool HI>
static hipError_t launch_tile(const RowsArgs &g, int keys, hipStream_t stream) {
    if (keys <= 256) return launch_tile_t<QC, 1, 4, HI>(g, stream);
    if (keys <= 512) return launch_tile_t<QC, 2, 4, HI>(g, stream);
    if (keys <= 1024) {
        [[maybe_unused]] const long long wgs = (long long)g.streams * g.a.n_head * ((g.t + RT_ROWS - 1) / RT_ROWS);
        if constexpr (QC > 1)
            if (wgs > 256) return launch_tile_t<QC, 4, 4, HI>(g, stream);
        return launch_tile_t<QC, 2, 8, HI>(g, stream);
    }
    return launch_tile_t<QC, 4, 8, HI>(g, stream);
}

// ---- Caches longer than a tile's registers ------------------------------------------------------------
// Key ranges of `span` keys over workgroups of four waves. The integer softmax needs the row maximum before the
// entries and their sum before p, so there are three walks over the keys, each forming the dots again (4 MFMAs
// a block and tile, less than keeping them would cost), one launch each over all ranges with the ranges' results in
// the workspace, and a last launch that adds the ranges' outputs:
//   k_long_scan<1> the extreme dots, <2> the sums: a wave takes blocks of keys with all WT row tiles of the group
//     (up to four), so the four waves' loads are of different keys;
//   k_long_pv the products with V: WT tiles side by side, 4 / WT waves to a tile, since a tile's sums are 64
//     registers for 64 channels (the others' loads of the same rows hit the L1).
// ALONE: k_long_pv walks all three times itself, where the rows alone give enough workgroups. A head dim above
// 128 takes a workgroup for each 64 channels (cg). 200 panels of 64 rows at 6,100 keys, head_dim 64: 139 us a call, by the
// kernel trace (which keeps the launches apart: 146 us) 14, 23, 58 and 5% of it. What the products' launch issues:
// per score 4 instructions to the table index, the lookup (LDS: 21 us in all, half of it bank conflicts), 6 for p and
// 3 for its digits (VALU: 32 us), 20 MFMAs a block (10 us), in chains that three waves a SIMD (160 VGPRs) overlap in part; K
// and V come a block ahead. A group's tile without rows leaves its wave idle: no limit, but not tried otherwise.
// Other shapes, a call: chunks of 256 causal rows with weights, 192 panels of 4,096 keys 203 us, 48 of 8,192 127;
// trees of 16 rows, 12 panels of 8,000 keys 38; of 64 rows and head_dim 256, 64 panels of 6,100 keys 374 (there the scans of
// four tiles spill: 2 registers in the first, 24 in the second, 37 at score shifts outside 32 to
// 60).
struct LongPlan {
    int tiles = 0, wt = 1, groups = 1;  // row tiles; of a group; groups
    int ng = 1, span = 0, cg = 1;        // key ranges, their keys; workgroups for the channels
};
struct LongScratch {
    int32_t *mm;    // [panels][rows][ng][2]: the largest and smallest dot of a range
    uint64_t *ps;   // [panels][rows][ng]: the sum of its entries
    int64_t *part;  // [panels][ng][rows][hd]: its sum p v
};

__host__ __device__ inline size_t al256(size_t x) { return (x + 255) / 256 * 256; }

__host__ __device__ inline LongScratch long_scratch(void *base, const LongPlan &p, size_t panels) {
    const size_t rows = panels * p.tiles * RT_ROWS;
    LongScratch s;
    s.mm = (int32_t *)base;
    s.ps = (uint64_t *)((char *)base + al256(rows * p.ng * 8));
    s.part = (int64_t *)((char *)s.ps + al256(rows * p.ng * 8));
    return s;
}

// One past the last key that the rows of tile group tg see.
__device__ __forceinline__ int group_keys(const RowsArgs &g, const StreamRows &R, const LongPlan &p, int tg) {
    const int keys = stream_keys(g, R), most = R.base + (tg + 1) * p.wt * RT_ROWS;
    return g.mask || keys < most ? keys : most;
}

template <int QC, int WT, bool HI, int PHASE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void k_long_scan(RowsArgs g, LongPlan pl, int panels, void *scratch) {
    extern __shared__ __attribute__((aligned(1024))) int8_t s_mem[];  // the table
    __shared__ uint64_t s_sum[4][WT][RT_ROWS];
    __shared__ int32_t s_mm[2][4][WT][RT_ROWS];
    const AttnArgs &a = g.a;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4;
    const int inner = pl.groups * pl.ng;
    const int L = blockIdx.x, panel = L / (8 * inner) * 8 + (L & 7);  // a panel's workgroups on one XCD
    const int in = (L >> 3) % inner;
    if (panel >= panels) return;
    const int tg = in % pl.groups, range = in / pl.groups;
    const int s = panel / a.n_head, h = panel - s * a.n_head, hd = a.hd;
    const StreamRows R = stream_rows(g, s);
    const int row0 = tg * WT * RT_ROWS;
    if (row0 >= R.count) return;
    const int keys = group_keys(g, R, pl, tg), k0 = range * pl.span;
    if (k0 >= keys) return;  // the ranges behind read no result of this one
    const int k1 = k0 + pl.span < keys ? k0 + pl.span : keys, last = a.exp_len - 1;
    int32_t *s_exp = (int32_t *)s_mem;
    if constexpr (PHASE == 2) load_table(a, s_exp, w, 4, lane);
    const size_t base = ((size_t)R.slot * a.n_head + h) * a.ctx_cap * hd;
    const Panel K(a.kc + base, a.ctx_cap, hd);
    const v4i zero = v4i{0, 0, 0, 0};
    v4i qf[WT][QC];
#pragma unroll
    for (int u = 0; u < WT; u++)
#pragma unroll
        for (int c = 0; c < QC; c++) {
            const int o = 64 * c + 16 * qg, row = row0 + RT_ROWS * u + ql;
            qf[u][c] = row < R.count && o < hd ? *(const v4i *)(a.q + (size_t)(R.first + row) * a.ldq + h * hd + o) : zero;
        }
    const int tiles = (R.count - row0 + RT_ROWS - 1) / RT_ROWS;  // of this group with rows (uniform)
    const LongScratch S = long_scratch(scratch, pl, panels);
    const int rows = pl.tiles * RT_ROWS, ranges = (keys + pl.span - 1) / pl.span;
    auto slot = [&](int u) { return ((size_t)panel * rows + row0 + RT_ROWS * u + ql) * pl.ng; };  // of a row's ranges

    int32_t dmax[WT], dmin[WT];
    uint64_t sum[WT];
#pragma unroll
    for (int u = 0; u < WT; u++) dmax[u] = INT32_MIN, dmin[u] = INT32_MAX, sum[u] = 0;
    if constexpr (PHASE == 2) {
#pragma unroll
        for (int u = 0; u < WT; u++)
            if (row0 + RT_ROWS * u + ql < R.count)
                for (int c = 0; c < ranges; c++) {
                    const int32_t x = S.mm[2 * (slot(u) + c)], y = S.mm[2 * (slot(u) + c) + 1];
                    dmax[u] = x > dmax[u] ? x : dmax[u];
                    dmin[u] = y < dmin[u] ? y : dmin[u];
                }
    }
    int64_t index[WT];
    if constexpr (PHASE == 2) {
#pragma unroll
        for (int u = 0; u < WT; u++) index[u] = RowIndex<HI>(a, dmax[u], dmin[u]).c;
        __syncthreads();  // the table
    }
    typedef v4i KRows[4][QC];
    int kb = k0 / 64 + w;
    auto k_load = [&](int b, KRows &x) {
#pragma unroll
        for (int c = 0; c < QC; c++) load_k<QC>(K, 64 * b, c, hd, 64 * b >= k1, lane, x);
    };
    RowSight sight[WT];
#pragma unroll
    for (int u = 0; u < WT; u++) sight[u] = row_sight(g, R, row0 + RT_ROWS * u + ql, qg, keys);
    auto step = [&](KRows &now, KRows &next) {
        k_load(kb + 4, next);
#pragma unroll
        for (int u = 0; u < WT; u++) {
            if (u >= tiles) break;
            const int t0 = row0 + RT_ROWS * u;  // the tile's first row
            int most = keys;
            if (!g.mask) most = R.base + t0 + RT_ROWS < keys ? R.base + t0 + RT_ROWS : keys;
            if (64 * kb >= most) continue;
            v4i D[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                D[t] = zero;
#pragma unroll
                for (int c = 0; c < QC; c++) D[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[t][c], qf[u][c], D[t], 0, 0, 0);
            }
            const int whole = g.mask ? R.base : R.base + t0 + 1;
            const bool all = 64 * kb + 64 <= (whole < most ? whole : most);
            const uint32_t ok = all ? 0u : sight_bits(sight[u], kb, lane, most);
            if constexpr (PHASE == 1) {
                block_extremes(D, all, ok, dmax[u], dmin[u]);
            } else {
                RowIndex<HI> ix(index[u]);
                block_entries<HI>(a, D, ix, s_exp, last, all, ok);
                sum[u] += block_sum(D);
            }
        }
        kb += 4;
        return 64 * kb < k1;
    };
    if (64 * kb < k1) {
        KRows x, y;
        k_load(kb, x);
        while (step(x, y) && step(y, x)) {}
    }
#pragma unroll
    for (int u = 0; u < WT; u++) {
        if constexpr (PHASE == 1) {
#pragma unroll
            for (int o = 16; o < 64; o <<= 1) {
                const int32_t x = __shfl_xor(dmax[u], o, 64), y = __shfl_xor(dmin[u], o, 64);
                dmax[u] = x > dmax[u] ? x : dmax[u];
                dmin[u] = y < dmin[u] ? y : dmin[u];
            }
            if (qg == 0) {
                s_mm[0][w][u][ql] = dmax[u];
                s_mm[1][w][u][ql] = dmin[u];
            }
        } else {
#pragma unroll
            for (int o = 16; o < 64; o <<= 1) sum[u] += __shfl_xor(sum[u], o, 64);
            if (qg == 0) s_sum[w][u][ql] = sum[u];
        }
    }
    __syncthreads();
    if (tid < WT * RT_ROWS && row0 + tid < R.count) {  // a thread per row
        const int u = tid >> 4, r = tid & 15;
        const size_t o = ((size_t)panel * rows + row0 + tid) * pl.ng + range;
        if constexpr (PHASE == 1) {
            int32_t x = s_mm[0][0][u][r], y = s_mm[1][0][u][r];
#pragma unroll
            for (int i = 1; i < 4; i++) {
                x = s_mm[0][i][u][r] > x ? s_mm[0][i][u][r] : x;
                y = s_mm[1][i][u][r] < y ? s_mm[1][i][u][r] : y;
            }
            S.mm[2 * o] = x;
            S.mm[2 * o + 1] = y;
        } else {
            S.ps[o] = s_sum[0][u][r] + s_sum[1][u][r] + s_sum[2][u][r] + s_sum[3][u][r];
        }
    }
}

template <int QC, int WT, bool HI, bool ALONE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(QC == 1 ? 3 : 2))) void k_long_pv(RowsArgs g, LongPlan pl, int panels, void *scratch) {
    constexpr int WK = 4 / WT, GC = QC > 2 ? 1 : QC;
    constexpr bool AHEAD = QC == 1;  // (above 64 channels the sums or K itself leave no registers for the next block)
    extern __shared__ __attribute__((aligned(1024))) int8_t s_mem[];
    __shared__ uint64_t s_sum[4][RT_ROWS];
    __shared__ int32_t s_mm[2][4][RT_ROWS];
    const AttnArgs &a = g.a;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, qg = lane >> 4, wt = w % WT, ks = w / WT;
    const int cgs = pl.cg, inner = pl.groups * pl.ng * cgs;
    const int L = blockIdx.x, panel = L / (8 * inner) * 8 + (L & 7);  // a panel's workgroups on one XCD
    int in = (L >> 3) % inner;
    if (panel >= panels) return;
    const int cg = in % cgs;
    in /= cgs;
    const int tg = in % pl.groups, range = in / pl.groups;
    const int s = panel / a.n_head, h = panel - s * a.n_head, hd = a.hd;
    const StreamRows R = stream_rows(g, s);
    if (tg * WT * RT_ROWS >= R.count) return;
    const int gkeys = group_keys(g, R, pl, tg), k0 = range * pl.span;
    if (!ALONE && k0 >= gkeys) return;  // the last launch reads no result of this one
    const int tile = tg * WT + wt, row = tile * RT_ROWS + ql, rows = pl.tiles * RT_ROWS;
    int keys = gkeys;
    if (!g.mask) keys = R.base + (tile + 1) * RT_ROWS < keys ? R.base + (tile + 1) * RT_ROWS : keys;
    if (tile * RT_ROWS >= R.count) keys = 0;  // a tile without rows walks nothing
    const int k1 = k0 + pl.span < keys ? k0 + pl.span : keys, last = a.exp_len - 1;
    int8_t *s_v = s_mem + 4096 * w;
    int32_t *s_exp = (int32_t *)(s_mem + 16384);  // the table, which the sums of the outputs take over
    load_table(a, s_exp, w, 4, lane);

    const size_t at = (size_t)R.slot * a.n_head + h, base = at * a.ctx_cap * hd;
    const Panel K(a.kc + base, a.ctx_cap, hd), V(a.vc + base, a.ctx_cap, hd);
    const v4i zero = v4i{0, 0, 0, 0};
    v4i qf[QC];
#pragma unroll
    for (int c = 0; c < QC; c++) {
        const int o = 64 * c + 16 * qg;
        qf[c] = row < R.count && o < hd ? *(const v4i *)(a.q + (size_t)(R.first + row) * a.ldq + h * hd + o) : zero;
    }
    const RowSight sight = row_sight(g, R, row, qg, keys);
    const int whole0 = g.mask ? R.base : R.base + tile * RT_ROWS + 1, whole = whole0 < keys ? whole0 : keys;
    // fn(the block, its dots, whether every row sees all of it, what the row sees)
    auto walk = [&](auto fn) {
        int kb = k0 / 64 + ks;
        v4i x[4][QC];
        auto k_load = [&](int b) {
#pragma unroll
            for (int c = 0; c < QC; c++) load_k<QC>(K, 64 * b, c, hd, 64 * b >= k1, lane, x);
        };
        if (AHEAD) k_load(kb);
        for (; 64 * kb < k1; kb += WK) {
            v4i D[4];
            if (!AHEAD) k_load(kb);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                D[t] = zero;
#pragma unroll
                for (int c = 0; c < QC; c++) D[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[t][c], qf[c], D[t], 0, 0, 0);
            }
            if (AHEAD) {  // the next block's K into the registers of this one's
                __builtin_amdgcn_sched_barrier(0);
                k_load(kb + WK);
            }
            const bool all = 64 * kb + 64 <= whole;
            fn(kb, D, all, all ? 0u : sight_bits(sight, kb, lane, keys));
        }
    };
    const LongScratch S = long_scratch(scratch, pl, panels);
    const size_t slot = ((size_t)panel * rows + row) * pl.ng;  // of the row's ranges
    const int ranges = (gkeys + pl.span - 1) / pl.span;

    int32_t dmax = INT32_MIN, dmin = INT32_MAX;
    if constexpr (ALONE) {
        walk([&](int, v4i (&D)[4], bool all, uint32_t ok) { block_extremes(D, all, ok, dmax, dmin); });
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
            const int32_t x = __shfl_xor(dmax, o, 64), y = __shfl_xor(dmin, o, 64);
            dmax = x > dmax ? x : dmax;
            dmin = y < dmin ? y : dmin;
        }
        if (WK > 1) {
            if (qg == 0) {
                s_mm[0][w][ql] = dmax;
                s_mm[1][w][ql] = dmin;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WK; i++) {
                const int32_t x = s_mm[0][wt + WT * i][ql], y = s_mm[1][wt + WT * i][ql];
                dmax = x > dmax ? x : dmax;
                dmin = y < dmin ? y : dmin;
            }
        }
    } else if (row < R.count) {
        for (int c = 0; c < ranges; c++) {
            const int32_t x = S.mm[2 * (slot + c)], y = S.mm[2 * (slot + c) + 1];
            dmax = x > dmax ? x : dmax;
            dmin = y < dmin ? y : dmin;
        }
    }
    const RowIndex<HI> ix(a, dmax, dmin);
    __syncthreads();  // the table
    uint64_t sum = 0;
    if constexpr (ALONE) {
        walk([&](int, v4i (&D)[4], bool all, uint32_t ok) {
            block_entries<HI>(a, D, ix, s_exp, last, all, ok);
            sum += block_sum(D);
        });
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
        if (WK > 1) {
            if (qg == 0) s_sum[w][ql] = sum;
            __syncthreads();
            sum = 0;
#pragma unroll
            for (int i = 0; i < WK; i++) sum += s_sum[wt + WT * i][ql];
        }
    } else if (row < R.count) {
        for (int c = 0; c < ranges; c++) sum += S.ps[slot + c];
    }
    const RowWeight weight(sum, a.softmax_p, row < R.count);
    v4i acc[GC][4][4];
#pragma unroll
    for (int c = 0; c < GC; c++)
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[c][k][i] = zero;
    uint64_t *mass = g.mass && cg == 0 ? g.mass + at * a.ctx_cap : nullptr;
    v4i vr[GC][4];  // arrives under the weights' arithmetic; one block ahead where K does
    auto v_load = [&](int b) {
#pragma unroll
        for (int c = 0; c < GC; c++) load_v(V, 64 * b, GC * cg + c, hd, 64 * b >= k1, lane, vr[c]);
    };
    if (AHEAD) v_load(k0 / 64 + ks);
    walk([&](int kb, v4i (&D)[4], bool all, uint32_t ok) {
        if (!AHEAD) v_load(kb);
        block_entries<HI>(a, D, ix, s_exp, last, all, ok);
        block_digits(D, weight.R, weight.sp, mass ? mass + 64 * kb : nullptr, k1 - 64 * kb, lane);
#pragma unroll
        for (int c = 0; c < GC; c++) {
#pragma unroll
            for (int u = 0; u < 4; u++) *(v4i *)(s_v + 1024 * u + 16 * lane) = vr[c][u];
            if (AHEAD) v_load(kb + WK);
            block_pv(s_v, D, lane, acc[c]);
        }
    });
    // A row's sums of one range, or the outputs themselves
    const double mo = a.out_s > 95 ? 0.0 : ldexp((double)a.out_m, -a.out_s);
    auto put = [&](int r, int ch, const int64_t (&x)[4]) {  // channels ch .. ch + 3 of row r
        if (ALONE) {
            uint32_t packed = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) packed |= (uint32_t)(uint8_t)(int8_t)attn_out_byte(x[e], mo, a.out_m, a.out_s) << (8 * e);
            *(uint32_t *)attn_out(a, R.first + r, h * hd + ch) = packed;
        } else {
            int64_t *o = S.part + (((size_t)panel * pl.ng + range) * rows + r) * hd + ch;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = x[e];
        }
    };
    if constexpr (WK == 1) {
        if (row < R.count) {
#pragma unroll
            for (int c = 0; c < GC; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int ch = 64 * (GC * cg + c) + 16 * i + 4 * qg;
                    int64_t x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = plane_sum(acc[c], i, e);
                    if (ch < hd) put(row, ch, x);
                }
        }
    } else {
        int64_t *s_acc = (int64_t *)s_exp;  // [WT][GC][16][RT_ACC], over the table
        __syncthreads();
        for (int i = tid; i < WT * GC * RT_ROWS * RT_ACC; i += 256) s_acc[i] = 0;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < GC; c++) {
            unsigned long long *to = (unsigned long long *)s_acc + ((wt * GC + c) * RT_ROWS + ql) * RT_ACC + 4 * qg;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) atomicAdd(to + 16 * i + e, (unsigned long long)plane_sum(acc[c], i, e));
        }
        __syncthreads();
        for (int i = tid; i < WT * GC * RT_ROWS * 16; i += 256) {
            const int q4 = i & 15, r = (i >> 4) & 15, c = (i >> 8) % GC, u = (i >> 8) / GC;
            const int ch = 64 * (GC * cg + c) + 4 * q4, out_row = (tg * WT + u) * RT_ROWS + r;
            if (ch >= hd || out_row >= R.count) continue;
            const int64_t *from = s_acc + ((u * GC + c) * RT_ROWS + r) * RT_ACC + 4 * q4;
            const int64_t x[4] = {from[0], from[1], from[2], from[3]};
            put(out_row, ch, x);
        }
    }
}

// The outputs from the ranges' sums: a thread per four channels.
__global__ __launch_bounds__(256) void k_rows_out(RowsArgs g, LongPlan pl, int panels, void *scratch) {
    const AttnArgs &a = g.a;
    const int rows = pl.tiles * RT_ROWS, quads = a.hd / 4;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t pr = i / quads;
    const int ch = 4 * (int)(i - pr * quads), panel = (int)(pr / rows), r = (int)(pr - (size_t)panel * rows);
    if (panel >= panels) return;
    const int s = panel / a.n_head, h = panel - s * a.n_head;
    const StreamRows R = stream_rows(g, s);
    if (r >= R.count) return;
    const int ranges = (group_keys(g, R, pl, r / (pl.wt * RT_ROWS)) + pl.span - 1) / pl.span;
    const LongScratch S = long_scratch(scratch, pl, panels);
    int64_t x[4] = {0, 0, 0, 0};
    for (int c = 0; c < ranges; c++) {
        const int64_t *p = S.part + (((size_t)panel * pl.ng + c) * rows + r) * a.hd + ch;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += p[e];
    }
    const double mo = a.out_s > 95 ? 0.0 : ldexp((double)a.out_m, -a.out_s);
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) packed |= (uint32_t)(uint8_t)(int8_t)attn_out_byte(x[e], mo, a.out_m, a.out_s) << (8 * e);
    *(uint32_t *)attn_out(a, R.first + r, h * a.hd + ch) = packed;
}

static LongPlan long_plan(const RowsArgs &g, int keys) {
    LongPlan p;
    p.tiles = (g.t + RT_ROWS - 1) / RT_ROWS;
    p.wt = p.tiles >= 3 ? 4 : p.tiles;
    p.groups = (p.tiles + p.wt - 1) / p.wt;
    p.cg = g.a.hd > 128 ? (g.a.hd + 63) / 64 : 1;
    // Ranges for about four workgroups a CU, at least two blocks a wave: three are resident, and where the caches are
    // partly empty (their ends' workgroups end at once) the rest is one round. Workgroups in all, 256, 512, 1,024 (this
    // rule), 2,048, 4,096, in us a call; caches of 8,192 places, all full, 6,100 and 3,000 keys in the mean:
    //   8 x 64 rows, 25 heads of 64      262 163 152 163 262   244 157 137 153 224   111 136  92  95 119
    //   16 x 64 rows, 25 heads of 64     321 321 284 258 284   301 301 273 219 258   148 148 212 135 152
    //   4 x 64 rows, 12 heads of 64       65  61  79  79  79    64  59  71  72  71    62  56  58  58  58
    //   32 x 16 rows, 12 heads of 64     120 120 143 152 161   106 106 117 122 135    54  54  75  70  76
    //   16 x 64 rows, 25 heads of 128    852 853 547 533 587   814 815 531 451 552   391 390 404 265 304
    //   8 x 64 rows, 25 heads of 256   2,668 1,369 1,164 1,246 1,480                  (full)
    // The best of them differs with the panels; this one is within 1.6 of it everywhere here, and 256 up to 2.3.
    constexpr long long LONG_WGS = 1024;
    const long long wgs = (long long)g.streams * g.a.n_head * p.groups;
    const int unit = 256, most = (keys + 2 * unit - 1) / (2 * unit);
    long long ng = LONG_WGS / wgs;
    ng = ng < 1 ? 1 : (ng > most ? most : ng);
    ng = ng < (keys + 65535) / 65536 ? (keys + 65535) / 65536 : ng;  // a wave's plane sums: at most 2^16 keys of 2^14
    p.span = (int)(((keys + ng - 1) / ng + unit - 1) / unit) * unit;
    p.ng = (keys + p.span - 1) / p.span;
    return p;
}

template <int QC, int WT, bool HI>
static hipError_t launch_long_t(const RowsArgs &g, const LongPlan &p, void *scratch, hipStream_t stream) {
    constexpr int GC = QC > 2 ? 1 : QC;
    const int panels = g.streams * g.a.n_head;
    const unsigned grid = (unsigned)((panels + 7) / 8 * 8) * p.groups * p.ng;
    const size_t table = (size_t)1024 * ((g.a.exp_len + 255) / 256), acc = WT < 4 ? (size_t)8 * WT * GC * RT_ROWS * RT_ACC : 0;
    auto run = [&](auto kernel, unsigned n, size_t lds) {
        const hipError_t e = allow_dynamic_lds((const void *)kernel, lds);
        if (e != hipSuccess) return e;
        launch_k(kernel, dim3(n), dim3(256), lds, stream, g, p, panels, scratch);
        return hipGetLastError();
    };
    const size_t lds = 16384 + (table > acc ? table : acc);
    hipError_t e;
    if (p.ng == 1) return run(k_long_pv<QC, WT, HI, true>, grid * p.cg, lds);
    if ((e = run(k_long_scan<QC, WT, HI, 1>, grid, 0)) != hipSuccess) return e;
    if ((e = run(k_long_scan<QC, WT, HI, 2>, grid, table)) != hipSuccess) return e;
    if ((e = run(k_long_pv<QC, WT, HI, false>, grid * p.cg, lds)) != hipSuccess) return e;
    const size_t quads = (size_t)panels * p.tiles * RT_ROWS * (g.a.hd / 4);
    launch_k(k_rows_out, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, g, p, panels, scratch);
    return hipGetLastError();
}

template <int QC, bool HI>
static hipError_t launch_long(const RowsArgs &g, const LongPlan &p, void *scratch, hipStream_t stream) {
    if (p.wt == 1) return launch_long_t<QC, 1, HI>(g, p, scratch, stream);
    if (p.wt == 2) return launch_long_t<QC, 2, HI>(g, p, scratch, stream);
    return launch_long_t<QC, 4, HI>(g, p, scratch, stream);
}

constexpr int ROWS_TASKS = (1 << 26) - 4;  // of k_rows in a launch, 64 threads each
constexpr int RT_KEYS = 2048;  // the most keys of a tile in one launch

static bool rows_hi(const AttnArgs &a) { return a.score_s >= 32 && a.score_s <= 60 && a.score_m != INT32_MIN; }

// Whether the MFMA forms take the shapes (a grid holds fewer than 2^32 threads), the alignments and the table.
static bool rows_mfma_ok(const RowsArgs &g) {
    const AttnArgs &a = g.a;
    const uintptr_t bits = (uintptr_t)a.q | (uintptr_t)a.kc | (uintptr_t)a.vc | (uintptr_t)a.exp_table | (uintptr_t)a.ldq | (uintptr_t)a.hd;
    const long long tiles = (g.t + RT_ROWS - 1) / RT_ROWS, panels = (long long)g.streams * a.n_head + 7;
    if (bits % 16 != 0 || a.exp_len > RT_TABLE) return false;
    if (panels * tiles >= 1ll << 23) return false;  // up to 512 threads a tile
    if (a.ctx_cap <= RT_KEYS) return true;
    const LongPlan p = long_plan(g, a.ctx_cap);
    return panels * p.groups * p.ng * p.cg < 1ll << 24 && panels * tiles * RT_ROWS * (a.hd / 4) < (1ll << 32) - 256;
}

// One causal row a stream: the decode kernels, which add up the weights too, where one launch of them serves (768
// row-heads of 1,024 keys 16.9 us, a tile each 36), and their split form for many row-heads over more keys than a tile
// holds. Else the forms for 16 rows: 12 row-heads of 2,000 keys 13.9 us, split 36; 768 of them 52 and 61; 12 of 8,000
// keys 27 (10 MB: 2.2 us; its four launches in a chain) and 79. Split form and walks at 192, 384, 516, 768 and 1,536 row-heads,
// all caches full:
//   head_dim 64,  2,100 keys    38 39    43 52    52 54    72 68   123 131
//   head_dim 64,  8,000 keys    83 90   123 148  160 227  226 313  441 621   (4,000 to 8,000: 190 and 241 at 768)
//   head_dim 32,  8,000 keys    58 63    91 88   113 116  146 145  282 278
//   head_dim 128, 8,000 keys   120 162  209 346  288 524  431 667  847 1,173
//   head_dim 256, 8,000 keys   237 454  443 831  623 1,849  846 2,470  1,692 4,999
// Above 64 channels the split form would win from fewer row-heads on than the 512 of this rule.
static bool rows_decode_ok(const RowsArgs &g) {
    const AttnArgs &a = g.a;
    const uintptr_t bits = (uintptr_t)a.q | (uintptr_t)a.kc | (uintptr_t)a.vc;
    if (g.t != 1 || g.mask || g.groups || !attend_split_ok(a.hd) || bits % 16 != 0) return false;
    if ((long long)g.streams * a.n_head >= 1ll << 22) return false;  // (up to 512 threads a row-head in a grid)
    return attend_split_one_launch(a.hd, a.ctx_cap, attend_split_plan(g.streams, a.n_head, a.ctx_cap)) || !rows_mfma_ok(g) ||
           (a.ctx_cap > RT_KEYS && (long long)g.streams * a.n_head >= 512);
}

size_t rows_workspace(const RowsArgs &g) {
    if (rows_decode_ok(g)) return attend_split_bytes(g.a, g.streams, attend_split_plan(g.streams, g.a.n_head, g.a.ctx_cap));
    if (g.a.ctx_cap <= RT_KEYS || !rows_mfma_ok(g)) return 0;
    const LongPlan p = long_plan(g, g.a.ctx_cap);
    if (p.ng == 1) return 0;
    const size_t panels = (size_t)g.streams * g.a.n_head;
    return (size_t)long_scratch(nullptr, p, panels).part + panels * p.ng * p.tiles * RT_ROWS * g.a.hd * 8;
}

// Past 1,024 keys a tile fills a CU, so three tiles and more of many panels walk the keys side by side instead (768
// panels of 64 rows at 1,400 keys: 147 us in tiles, 103 in one launch of three walks; at 700 keys 60 and 58, 192
// panels 19 and 32).
template <int QC, bool HI>
static hipError_t launch_mfma(const RowsArgs &g, void *workspace, hipStream_t stream) {
    const LongPlan p = long_plan(g, g.a.ctx_cap);
    const bool walks = g.a.ctx_cap > RT_KEYS || (g.a.ctx_cap > 1024 && p.tiles >= 3 && p.ng == 1);
    return walks ? launch_long<QC, HI>(g, p, workspace, stream) : launch_tile<QC, HI>(g, g.a.ctx_cap, stream);
}

// Without the workspace that a shape's fast form needs: the row form.
hipError_t launch_rows(const RowsArgs &g, void *workspace, hipStream_t stream) {
    if (g.streams <= 0 || g.t <= 0 || g.a.n_head <= 0) return hipSuccess;
    const bool fast = workspace || rows_workspace(g) == 0;
    if (fast && rows_decode_ok(g)) {
        AttnArgs a = g.a;
        a.keys = g.ctx;
        a.count = g.count;
        a.mass = g.mass;
        return launch_attend_split(a, g.streams, attend_split_plan(g.streams, a.n_head, a.ctx_cap), workspace, stream);
    }
    if (fast && rows_mfma_ok(g)) {
        const bool hi = rows_hi(g.a);
        if (g.a.hd <= 64) return hi ? launch_mfma<1, true>(g, workspace, stream) : launch_mfma<1, false>(g, workspace, stream);
        if (g.a.hd <= 128) return hi ? launch_mfma<2, true>(g, workspace, stream) : launch_mfma<2, false>(g, workspace, stream);
        return hi ? launch_mfma<4, true>(g, workspace, stream) : launch_mfma<4, false>(g, workspace, stream);
    }
    // as many streams in a launch as a grid holds threads (fewer than 2^32) for: the batch may bring more
    const int rows = g.t * g.a.n_head, most = ROWS_TASKS / rows < 1 ? 1 : ROWS_TASKS / rows;
    for (int s0 = 0; s0 < g.streams; s0 += most) {
        const int tasks = (g.streams - s0 < most ? g.streams - s0 : most) * rows;
        launch_k(k_rows, dim3((tasks + 3) / 4), dim3(256), 0, stream, g, s0, tasks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace hs
