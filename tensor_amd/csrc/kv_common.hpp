// What the launches on the paged int8 cache of keys and values share: its layout, the batch's geometry and the rounding to codes.
#pragma once

#include "common.hpp"

namespace ohip {

constexpr int KV_BLOCK = 64;  // tokens of a page: they share a scale for each head

// Scales below this count as 0: their codes are all 0. It keeps the exact comparisons of code_of clear of the smallest numbers.
constexpr float KV_LEAST_SCALE = 0x1p-100f;

// A page of one head is 4 * chunks tiles of 1 KiB for the keys and as many for the values, chunks = ceil(head_dim / 64), each the
// operand of one 16x16x64 matrix instruction in lane order: a lane's 16 bytes at 16 * lane.
//   keys   tile [dims / 64][tokens / 16], row = token % 16, contraction = dim % 64
//   values tile [dims / 16], row = dim % 16, contraction = token, in the order that the scores' lanes hold the tokens:
//          slot 16 g + 4 t + r is token 16 t + 4 g + r, so that the weights of a row go into the second product without leaving
//          their lanes
// Both are loaded as whole contiguous KiB. Dims behind head_dim are 0.
struct KvView {
    int8_t *k, *v;
    float *ks, *vs;  // [pages][heads]
    int heads, dim, n_pages, chunks;
    __host__ __device__ size_t head_bytes() const { return (size_t)chunks * 4096; }
    __device__ size_t at(int page, int head) const { return ((size_t)page * heads + head) * head_bytes(); }
};
// byte of (token, dim) in a page's head
__host__ __device__ inline int kv_key_byte(int token, int dim) {
    return ((dim >> 6) * 4 + (token >> 4)) * 1024 + ((dim >> 4) & 3) * 256 + (token & 15) * 16 + (dim & 15);
}
__host__ __device__ inline int kv_value_byte(int token, int dim) {
    return (dim >> 4) * 1024 + ((token >> 2) & 3) * 256 + (dim & 15) * 16 + (token >> 4) * 4 + (token & 3);
}

struct KvBatch {
    int n_seqs, n_tokens, max_pages;
    const int32_t *starts, *lengths, *pages;
};

// One sequence of a batch as the kernels see it: what a table that is wrong could say is cut to what the buffers hold.
struct KvSeq {
    int index;
    int begin, count;  // its rows
    int length;        // tokens, with those of the rows
    int first;         // position of its first row (below 0: the batch says more rows than tokens)
    int tile;          // of the sequence (below 0: of none)
    int all;           // tiles of all sequences (-1: more than 64 of them, not counted)
};

// The sum over this lane and those below it.
__device__ __forceinline__ int lanes_below(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // a row of 16 lanes: one to the right,
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // two,
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // four,
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // eight
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // the last of rows 0 and 2 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // the last of row 1 into rows 2 and 3
    return v;
}

// Work is dealt to tiles of UNIT rows of a sequence (mul rows for each of `starts`; BLOCKS: to the blocks of 64 positions that its rows lie
// in) without a list of them, by the lanes of a wave, and what is to be known of the sequence that is found comes along.
// Up to 64 sequences: a lane counts the tiles of one, and a sum over the lanes says whose the tile is. More: sequence i's tiles
// begin at starts[i] * mul / UNIT + SLACK * i, which leaves each at least as many as it needs (ceil(n / UNIT) <= floor difference + 1, and
// one more where blocks are aligned to positions), and a load for each 64-fold of sequences finds the largest i whose tiles begin at or
// before the tile. The first way leaves no tiles empty but the grid's last ones: workgroups are handed to the shader engines in
// turn, and empty ones among them left some engines with one more than others (32 sequences of 5 query heads to a key head, 8 key heads,
// one workgroup a compute unit: 65 us, with 4 query heads 47).
template <int UNIT, bool BLOCKS, bool LENGTHS>
__device__ __forceinline__ KvSeq kv_locate(const int32_t* starts, const int32_t* lengths, int n, int limit, int mul, int tile) {
    constexpr int SLACK = BLOCKS ? 2 : 1;
    const int lane = (int)(threadIdx.x & 63);
    int lo = 0, all = -1;
    const bool few = n <= 64;
    for (;;) {
        const int step = (n + 63) >> 6, i = lane * step, at = lo + min(i, n - 1);
        const int from = min(max(starts[at], 0), limit), count = min(max(starts[at + 1], from), limit) - from;
        int length = 0;
        if constexpr (LENGTHS) length = max(lengths[at], 0);
        int base, k;
        if (few) {
            int tiles = BLOCKS ? ((length - 1) >> 6) - ((length - count) >> 6) + 1 : (int)((unsigned)(count * mul + UNIT - 1) / UNIT);
            if (i >= n || count == 0) tiles = 0;
            base = lanes_below(tiles);
            all = __builtin_amdgcn_readlane(base, 63);
            base -= tiles;
            const unsigned long long mine = __ballot(tiles > 0 && base <= tile);
            k = mine ? 63 - __builtin_clzll(mine) : 0;
            if (!mine) base = tile + 1;  // (no sequence has rows)
        } else {
            base = (int)((unsigned)(from * mul) / (unsigned)UNIT) + SLACK * at;
            k = max(__popcll(__ballot(i < n && base <= tile)), 1) - 1;
        }
        if (step == 1) {
            KvSeq s;
            s.index = __builtin_amdgcn_readfirstlane(lo + k);
            s.begin = __builtin_amdgcn_readlane(from, k);
            s.count = __builtin_amdgcn_readlane(count, k);
            s.length = __builtin_amdgcn_readlane(length, k);
            s.first = s.length - s.count;
            s.tile = tile - __builtin_amdgcn_readlane(base, k);
            s.all = all;
            return s;
        }
        lo += k * step;
        n = min(step, n - k * step);
    }
}

// |x| of a finite value, 0 for an infinity or NaN: what a scale is found from.
__device__ __forceinline__ float finite_size(float x) {
    const float a = __builtin_fabsf(x);
    return a < __builtin_inff() ? a : 0.f;
}
// The largest finite size of N values: compared as integers, which order sizes as floats do and have what is not finite above all others,
// so that a value costs a mask and half a comparison; where something is not finite, once more by finite_size.
template <int N>
__device__ __forceinline__ float largest_size(const float (&x)[N]) {
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
    if (most < 0x7f800000u) return __uint_as_float(most);
    float finite = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) finite = fmaxf(finite, finite_size(x[e]));
    return finite;
}
__device__ __forceinline__ float scale_of(float most) {
    const float s = __fdiv_rn(most, 127.f);
    return s < KV_LEAST_SCALE ? 0.f : s;
}

// x / s rounded half away from zero, at most 127, exactly (NaN: 0). The product with the rounded reciprocal is off by less than
// 2^-15, so its rounding is off by one at most; whether it is tells the sign of |x| - (c -+ 1/2) s, which one fused multiply-add
// has right. s is at least KV_LEAST_SCALE (then no result of it underflows), inv = 1 / s.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    const float a = fminf(__builtin_fabsf(x), __fmul_rn(s, 128.f));  // (an infinity; NaN becomes 128 steps: taken out below)
    float c = __builtin_floorf(__fadd_rn(__fmul_rn(a, inv), 0.5f));
    if (__fmaf_rn(__fadd_rn(c, -0.5f), -s, a) < 0.f) c = __fadd_rn(c, -1.f);
    else if (__fmaf_rn(__fadd_rn(c, 0.5f), -s, a) >= 0.f) c = __fadd_rn(c, 1.f);
    const int i = min((int)c, 127);
    return x == x ? (x < 0.f ? -i : i) : 0;
}
// The four codes of a word, and whether one of them may be wrong: then code_of has to find them. c = rint(x / s), the quotient off by
// less than 2^-15, is right where |x - c s| < s / 2; one fused multiply-add has that difference, rounded, and a rounding does not pass s / 2.
// (Not below s / 2: the middle between two codes, a code that is off by one, an infinity, NaN.) Eight instructions a code with their
// packing, where code_of is twenty: one token for each of 48 sequences appended in 5.6 us for 6.9, 4096 rows of 2816 rounded in 13.0 for 15.0.
struct Coder {
    float s, inv, half;
    __device__ explicit Coder(float scale) : s(scale) {
        inv = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
        half = scale > 0.f ? __fmul_rn(scale, 0.5f) : __builtin_inff();
    }
    __device__ __forceinline__ int word(float x, float y, float z, float w, bool& doubtful) const {
        const float v[4] = {x, y, z, w};
        unsigned c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = __builtin_rintf(__fmul_rn(v[e], inv));
            doubtful |= !(__builtin_fabsf(__fmaf_rn(-q, s, v[e])) < half);
            c[e] = (unsigned)(int)q;
        }
        const unsigned low = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), high = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0c);
        return (int)(low | high);
    }
    __device__ __forceinline__ int exact(float x) const { return s > 0.f ? code_of(x, s, inv) & 0xff : 0; }
    __device__ __forceinline__ int exact_word(float x, float y, float z, float w) const {
        return exact(x) | exact(y) << 8 | exact(z) << 16 | exact(w) << 24;
    }
};

// kv_cache.hip
hipError_t run_kv_append(const KvView& c, const KvBatch& b, const float* k, size_t k_stride, const float* v, size_t v_stride, hipStream_t stream);
hipError_t run_kv_read(const KvView& c, const KvBatch& b, float* k, float* v, hipStream_t stream);

// kv_attend.hip
int kv_attend_tiles(int n_tokens, int n_seqs, int group);
struct KvPlan {
    bool staged;
    int waves, splits;
};
KvPlan kv_attend_plan(int n_tokens, int n_seqs, int group, int heads, int chunks, bool extra, int max_pages);
hipError_t run_kv_attend(const KvView& c, const KvBatch& b, const float* q, size_t q_stride, float* out, int q_heads, float scale, float cap,
                         const float* slopes, int causal, int window, const KvPlan& plan, void* workspace, hipStream_t stream);

}  // namespace ohip
