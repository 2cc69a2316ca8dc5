// The device pieces that the attention kernels share: the score and output rules, wave reductions and the
// digit-plane products of the weights with V.
#pragma once

#include "intmath.h"
#include "launch.h"

namespace hs {

constexpr int64_t SCORE_LIMIT = (int64_t)1 << 40;  // gpt2/mod.rs:119

// A table that the waves copied to LDS straight is there for the whole workgroup. Such loads are no LDS operations to a barrier, which
// waits for those alone (lgkmcnt): each wave waits for its own.
__device__ __forceinline__ void table_there() {
    wait_vmcnt<0>();
    __syncthreads();
}

// ---- wave reductions (wave64) -------------------------------------------------------------

__device__ __forceinline__ int64_t wave_max64(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        int64_t u = __shfl_xor(v, o, 64);
        v = u > v ? u : v;
    }
    return v;
}

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ int32_t dot_key(const int *q4, const int8_t *k, int hd) {
    int32_t s = 0;
    const int *k4 = (const int *)k;
    for (int c = 0; c < hd / 4; c++) s = __builtin_amdgcn_sdot4(q4[c], k4[c], s, false);
    return s;
}

// The keys of a decode row whose count is n: one at least, and never past the cache. (Compared unsigned: as an int
// a count from 2^31 on would be negative, one key.)
__device__ __forceinline__ int decode_keys(const AttnArgs &a, uint32_t n) {
    return n < 1 ? 1 : (n > (uint32_t)a.ctx_cap ? a.ctx_cap : (int)n);
}

// score = clamp(rescale(dot, m, s), +-2^40): |dot| <= hd 2^14 <= 2^22, so |dot m| < 2^53 and one
// multiply-add and an arithmetic shift are exact (a shift of 63 or more gives 0). With s >= 13
// the score stays within +-2^40 and the clamp is a no-op.
__host__ __device__ inline bool attn_noclamp(const AttnArgs &a) { return a.score_s >= 13; }

// The attention output byte clamp(rescale(v, m, s), +-127) for an exact |v| < 2^53 (the sum of
// p v): y = v m 2^-s + 1/2 in double (mo = m 2^-s, exact; v exact; one rounding in the fused
// multiply-add, relative 2^-53). When |y| >= 256 the clamp decides; when y lies at least 2^-30
// from an integer floor(y) is exact (|y| < 256: the error is below 2^-45); else the i128 rule.
__device__ __forceinline__ int32_t attn_out_byte(int64_t v, double mo, int32_t m, int s) {
    const double y = fma((double)v, mo, 0.5);
    const double f = __builtin_amdgcn_fract(y);
    if (fabs(y) >= 256.0 || fabs(f - 0.5) <= 0.5 - 0x1p-30) return (int32_t)fmin(fmax(y - f, -127.0), 127.0);
    return (int32_t)clamp128(rescale_full(v, m, s), -127, 127);
}

template <bool NOCLAMP>
__device__ __forceinline__ int64_t attn_score(const AttnArgs &a, int32_t dot) {
    const int s_eff = a.score_s < 63 ? a.score_s : 63;
    const int64_t s_half = s_eff ? (int64_t)1 << (s_eff - 1) : 0;
    const int64_t r = ((int64_t)dot * a.score_m + s_half) >> s_eff;
    return NOCLAMP ? r : clamp64(r, -SCORE_LIMIT, SCORE_LIMIT);
}

// ---- The pieces of the one-launch decode kernels ---------------------------------------------------
// Sum p v of one query row is a product of a 64-channel x 64-key matrix with p, and p is four
// balanced i8 digits (the bytes of p + 0x80808080, xor 0x80): one v_mfma_i32_16x16x64_i8 takes 16
// channels x 64 keys against the four digit planes as four of its columns (the other twelve
// repeat them), so a block of 64 keys is 4 MFMAs where 24-bit multiplies took 192 VALU
// instructions a wave, and the sums need no butterfly over the lanes.
// A block's V rows lie in LDS as dense rows of 16 NC bytes (NC = 4: head dims from 64 on, in groups
// of 64 channels; below that one group of hd), 16-byte chunk c of row r at slot NC r + (c ^ vsw(r));
// the V^T operand comes by transposing reads (as in k_attend_short), whose operand byte 4 t + e of
// lane group g holds key 16 t + 4 g + e. `mem` is 1 KiB of the wave.
template <int NC>
__device__ __forceinline__ int vsw(int r) {
    return NC == 4 ? ((r >> 1) ^ (r >> 3)) & 3 : NC == 2 ? (r >> 2) & 1 : 0;
}

// Lane l's p of key l to the digit operand of the block.
__device__ __forceinline__ v4i decode_pv_digits(int8_t *mem, uint32_t p, int lane) {
    const uint32_t q = (p + 0x80808080u) ^ 0x80808080u;
    int8_t *w = mem + 16 * ((lane >> 2) & 3) + 4 * (lane >> 4) + (lane & 3);
#pragma unroll
    for (int k = 0; k < 4; k++) w[64 * k] = (int8_t)(q >> (8 * k));
    return *(const v4i *)(mem + 64 * (lane & 3) + 16 * (lane >> 4));
}
template <int NC>
__device__ __forceinline__ void decode_pv_block(const int8_t *sv, const v4i &pf, int lane, v4i *acc) {
    const int ql = lane & 15, qg = lane >> 4;
    const int tr_k = ql >> 1, tr_h = ql & 1;
    const int key0 = 16 * (tr_k >> 2) + 4 * qg + (tr_k & 3);
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int8_t *p0 = sv + (NC * key0 + (c ^ vsw<NC>(key0 & 15))) * 16 + 8 * tr_h;
        const v2i r0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)p0);
        const v2i r1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(p0 + 32 * 16 * NC));
        acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v4i{r0[0], r0[1], r1[0], r1[1]}, pf, acc[c], 0, 0, 0);
    }
}

// acc[c][e] of lane l holds channel 16 c + 4 (l / 16) + e of plane l % 16 (< 4): to [plane][64] in mem.
template <int NC>
__device__ __forceinline__ void decode_pv_store(int8_t *mem, int lane, const v4i *acc) {
    if ((lane & 15) < 4) {
#pragma unroll
        for (int c = 0; c < NC; c++) *(v4i *)(mem + 256 * (lane & 15) + 64 * c + 16 * (lane >> 4)) = acc[c];
    }
}
// The planes' sum of channel ch: below 2^24 per plane, |sum| <= 1,024 2^30 2^7 < 2^53.
__device__ __forceinline__ int64_t decode_pv_sum(const int8_t *mem, int ch) {
    const int32_t *m = (const int32_t *)mem + ch;
    return (int64_t)m[0] + (int64_t)m[64] * 256 + (int64_t)m[128] * 65536 + (int64_t)m[192] * 16777216;
}

// The extreme values over the wave.
__device__ __forceinline__ void wave_min_max(int32_t &mn, int32_t &mx) {
    butterfly<64>([&](auto st) {
        constexpr int S = decltype(st)::value;
        const int32_t u = lane_move<S>(mn), v = lane_move<S>(mx);
        mn = u < mn ? u : mn;
        mx = v > mx ? v : mx;
    });
}
__device__ __forceinline__ uint64_t wave_sum_dpp(uint64_t v) {
    butterfly<64>([&](auto st) { v += (uint64_t)lane_move64<decltype(st)::value>((int64_t)v); });
    return v;
}

}  // namespace hs
