// Attention over the paged int8 cache (layout: kv_common.hpp).
//
//   t_j = scale * q . k_j      k_j = key codes * the page's key scale        t_j = cap * tanh(t_j / cap)      t_j -= slope * |p - j|
//   o   = sum_j exp(t_j - m) v_j / sum_j exp(t_j - m)
//
// Both products run on the int8 matrix cores, on the cache's bytes as they are. The float operands go in as fixed point of three
// 8-bit digits: a query row in units of 2^-22 of its largest element's binade, the weights exp(t_j - m) in units of 1 / WEIGHT_UNITS
// of the largest weight that the row has in the page. Digit products and their sums are exact in 32 bits, so a score is off by what
// rounding q to 23 bits makes of it, and a page's share of o by half a unit times the code for each token. Where o is large in these units,
// that is what sums in 32-bit floats are off by. Where it is not -- the tokens that have the weight have values near 0, and o is what the
// others make of theirs -- the digits behind follow (`finer` in the kernel). (Half floats would need a second operand for the bits behind
// the 11th, and the bytes of the cache converted for every row tile: two products at half the rate and five vector instructions for four
// bytes, against three products at the full rate on bytes that are only loaded.)
//
// A wave owns 16 query rows: the tokens of a sequence times the query heads that share a key head. The scores come transposed (keys x
// rows), so a row's statistics and scale factors live in the lanes of its column, and the weights are already where the second
// product wants them; nothing crosses lanes but the row maxima. The running maximum and sum are fp32, one rescaling a page.
#include "kv_common.hpp"

namespace ohip {

// tanh(x) / x as a polynomial of x^2, the smallest largest relative error for |x| < 1/2: 2^-26.
constexpr int TANH_TERMS = 5;
constexpr double TANH_TERM[TANH_TERMS] = {0.9999999868718333, -0.3333306939402176, 0.13324779317606145, -0.05298607529097958, 0.0171350066330358};

struct Cap {
    float cap;               // cap * log2(e), 0: none
    float half[TANH_TERMS];  // that times the terms of tanh below 1/2
};

struct AttendArgs {
    KvView c;
    KvBatch b;
    const float* q;
    size_t q_stride;
    float* out;
    int q_heads, group;
    float scale;  // with cap: scale / cap, else scale * log2(e)
    Cap cap;
    const float* slopes;
    int causal, window;
    int tiles, splits;
    float *part_o, *part_ml;  // of a split: [split][row][dim], [split][row][2] with row = token * q_heads + head
};

// What a weight of 1 is as a whole number: a little below what three signed digits hold and, with the 0x8080 that makes them, below 2^23.
constexpr float WEIGHT_UNITS = 8350000.f;

// A row is made finer whose largest element is below this many units of its weights times a code of 1. The roundings, 0.29 units each, are 293
// units together for 64 tokens with codes of 127: 2^-16.8 of that element, and 2^-18.6 with codes of normal values. Ordinary rows are ten times
// above the limit: one token with the largest weight and a code of 40 is.
constexpr float ROUGH = 0x1p25f;

constexpr float LOG2E = 1.44269504088896340736f;

// Over the four lanes that share a column, 16 apart. (The exchanges put both halves, or both rows of 16, of a register beside each
// other in two; no LDS.)
__device__ __forceinline__ float quad_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __fadd_rn(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __fadd_rn(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// times * tanh(x) / x for |x| < 1/2, of x * x; terms: TANH_TERM times that
__device__ __forceinline__ float tanh_of_half(float y, const float (&terms)[TANH_TERMS]) {
    float s = terms[TANH_TERMS - 1];
#pragma unroll
    for (int n = TANH_TERMS - 2; n >= 0; --n) s = __fmaf_rn(y, s, terms[n]);
    return s;
}
// tanh of |x| >= 1/2: 1 - 2 / (exp(2 |x|) + 1), which loses the bits of smaller ones. (The reciprocal is that of the hardware, off by one unit
// in the last place at most: a division is ten instructions, a third of all here.)
__device__ __forceinline__ float tanh_of_more(float x) {
    const float e = fast_exp2(__fmul_rn(__builtin_fabsf(x), 2.f * LOG2E));
    return __builtin_copysignf(__fmaf_rn(-2.f, __builtin_amdgcn_rcpf(__fadd_rn(e, 1.f)), 1.f), x);
}

// Three signed digits of four fixed-point numbers (u = number + 0x8080 in the low 24 bits): u's low two bytes less 128, and the third.
__device__ __forceinline__ void split_digits(const unsigned (&u)[4], int& low, int& mid, int& high) {
    const unsigned ab = __builtin_amdgcn_perm(u[1], u[0], 0x05010400);  // a0 b0 a1 b1
    const unsigned cd = __builtin_amdgcn_perm(u[3], u[2], 0x05010400);
    low = (int)(__builtin_amdgcn_perm(cd, ab, 0x05040100) ^ 0x80808080u);
    mid = (int)(__builtin_amdgcn_perm(cd, ab, 0x07060302) ^ 0x80808080u);
    const unsigned a2b2 = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0602), c2d2 = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0602);
    high = (int)__builtin_amdgcn_perm(c2d2, a2b2, 0x05040100);
}

typedef ohip_v4i v4i;
__device__ __forceinline__ v4i mma(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
// (high * 256 + mid) * 256 + low: the first step is below 2^31 for 256 dims
__device__ __forceinline__ float join_digits(int high, int mid, int low) { return __fmaf_rn((float)((high << 8) + mid), 256.f, (float)low); }

template <int KC>
struct Queries {
    v4i digit[3][KC];  // high, mid, low
    float unit;        // what 1 stands for (NaN: the row holds a NaN or an infinity)
};

// A lane's share of its row: 16 dims of every 64; `negative`: of the row times -1 (the units are never negative).
template <int KC>
__device__ __forceinline__ void load_queries(Queries<KC>& q, const float* __restrict__ row, int dim, bool whole, bool negative) {
    const int g = (int)(threadIdx.x >> 4) & 3;
    float x[KC][16];
    float most = 0.f;
    bool odd = false;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        const int d0 = c * 64 + g * 16;
        if (whole) {  // (rows at 16 bytes, whole quads)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float4 f = {0.f, 0.f, 0.f, 0.f};
                if (d0 + e < dim) f = *reinterpret_cast<const float4*>(row + d0 + e);
                x[c][e] = f.x, x[c][e + 1] = f.y, x[c][e + 2] = f.z, x[c][e + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[c][e] = d0 + e < dim ? row[d0 + e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float a = __builtin_fabsf(x[c][e]);
            odd |= !(a < __builtin_inff());
            most = fmaxf(most, a);
        }
    }
    most = quad_max(odd ? __builtin_inff() : most);
    odd = !(most < __builtin_inff());
    // units of 2^(e - 22), most in [2^e, 2^(e + 1)) but for the binade's last part, which would have more of them than three signed digits
    // (127 * 2^16 + 127 * 2^8 + 127): it counts as the next one's. (A row below 2^-100 counts as 0.)
    const int e = (int)(__float_as_uint(__fmul_rn(most, 1.0041f)) >> 23) - 127;
    const bool none = odd || e < -100;
    const float size = none ? 0.f : __uint_as_float((unsigned)(127 + 22 - e) << 23), per = negative ? -size : size;
    q.unit = odd ? __builtin_nanf("") : none ? 0.f : __uint_as_float((unsigned)(127 - 22 + e) << 23);
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            unsigned u[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u[r] = (unsigned)((none ? 0 : (int)__builtin_rintf(__fmul_rn(x[c][4 * t + r], per))) + 0x8080);
            }
            int lo, mi, hi;
            split_digits(u, lo, mi, hi);
            q.digit[2][c][t] = lo, q.digit[1][c][t] = mi, q.digit[0][c][t] = hi;
        }
}

template <int KC>
struct Running {
    float o[4 * KC][4];  // [16 dims][lane group's four]
    float m, l;          // maximum (log2), this lane's share of the sum
    float second;        // the largest maximum of any step but the one that has m
};
// Of the steps that a wave takes, its rows together: the largest value scale (as an integer) and which of them raised the maximum of a row,
// a bit each, the last for all from the 64th on. In scalar registers, as there is no vector register to spare; one vector instruction a step
// for `second`.
struct Steps {
    unsigned scale;
    unsigned long long raised;
    int now;
    __device__ float unit() const { return __fmul_rn(__uint_as_float(scale), 1.f / WEIGHT_UNITS); }  // what a unit of a weight is of o, at the most
    __device__ bool raises(int step) const { return (raised >> min(step, 63)) & 1; }
};
// For REST of attend_pages: the lanes of which a unit is more than `least` of o get the digits behind the first three (level 1), six or nine.
struct Finer {
    float least;
    int level;
};

// What a step of NP pages has beside their codes: the scales, and the positions of their first tokens.
template <int NP>
struct Pages {
    float k_scale[NP], v_scale[NP];
    int first[NP];
    bool all;  // all of them are pages of the pool
};
// What a lane's row sees, [lo, hi), and where it is itself.
struct RowView {
    int lo, hi, p;
    float slope;
    float rise[4][4];  // slope * distance to the page's last token, below 0, of a lane's scores
};

// NP pages into a wave's 16 rows. key(page, tile) and value(page, tile): the lane's 16 bytes of a tile; keys_done and values_done: called
// when the last of them is used. whole: every row sees all of them; behind: none of their
// tokens is behind a row. Two pages at a time share the conversions of the second product's sums and the rescaling of o, a quarter of the vector
// instructions of one: the weights go in as multiples of the pages' value scales, in units of 1 / WEIGHT_UNITS of the largest such product.
// REST: the pages are in, and what the rounding of their weights has left out follows, three more digits.
template <int KC, int EXTRA, int NP, bool REST, typename Key, typename Value, typename KeysDone, typename ValuesDone>
__device__ __forceinline__ void attend_pages(Running<KC>& s, const Queries<KC>& q, const Key& key, const Value& value, const KeysDone& keys_done,
                                             const ValuesDone& values_done, const Pages<NP>& at, float factor, const Cap& cap, const RowView& row,
                                             bool whole, bool behind, Steps& steps, const Finer& finer = {}) {
    const int g = (int)(threadIdx.x >> 4) & 3;
    // scores (log2) are t * unit_of + away; without cap and slopes the product is left to the subtraction of the maximum
    float t[NP][4][4], most_of[NP], unit_of[NP], away = 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const float unit = __fmul_rn(factor, at.k_scale[p]);
        unit_of[p] = EXTRA == 0 ? unit : 1.f;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            v4i a[3] = {};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const v4i k = key(p, c * 4 + kt);
#pragma unroll
                for (int n = 0; n < 3; ++n) a[n] = mma(k, q.digit[n][c], a[n]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = join_digits(a[0][r], a[1][r], a[2][r]);
                t[p][kt][r] = EXTRA == 0 ? x : __fmul_rn(x, unit);  // (with a cap too here, in the shadow of the products)
            }
        }
        if constexpr (EXTRA != 0) {
            // In a page whose tokens are no further than the rows (`behind`) the distance is that of the page's last token, the same for all,
            // which joins the maximum, and what a token is in front of it, added with the score's last product. (Relative to the nearest
            // token the sums are as precise as those of the tokens that count. Over 64 dims there are no registers for it, and without a cap
            // it is no faster. Six prompts of up to 1900 tokens, cap, slopes, window 512, 16 heads of 64: 56.3 -> 52.2 us with the cap's polynomial.)
            static_assert(NP == 1, "one page has one `away`");
            // last(i, x, f): score i is x * f, less its slope
            const auto scores = [&](const auto& last) {
                float (&x)[4][4] = t[p];
                if (EXTRA == 1 || cap.cap != 0.f) {
                    // Most scores are far below the cap: a third of the instructions for a page where all are below half of it. The vote counts
                    // slots that no row sees, whatever they hold: a score's bits are the same either way.
                    float far = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) far = fmaxf(far, __builtin_fabsf(x[i >> 2][i & 3]));
                    if (__all(far < 0.5f)) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            x[i >> 2][i & 3] = last(i, x[i >> 2][i & 3], tanh_of_half(__fmul_rn(x[i >> 2][i & 3], x[i >> 2][i & 3]), cap.half));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float y = x[i >> 2][i & 3], more = tanh_of_more(y), half = tanh_of_half(__fmul_rn(y, y), cap.half);
                            const bool less = __builtin_fabsf(y) < 0.5f;
                            x[i >> 2][i & 3] = last(i, less ? y : more, less ? half : cap.cap);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i >> 2][i & 3] = last(i, x[i >> 2][i & 3], 1.f);
                }
            };
            if constexpr (EXTRA == 1) scores([](int, float x, float f) { return __fmul_rn(x, f); });
            else if (KC == 1 && behind && cap.cap != 0.f) {
                away = __fmul_rn(-row.slope, (float)(row.p - (at.first[p] + KV_BLOCK - 1)));
                scores([&](int i, float x, float f) { return __fmaf_rn(x, f, row.rise[i >> 2][i & 3]); });
            } else {
                const float to = (float)(row.p - at.first[p] - 4 * g);
                scores([&](int i, float x, float f) {
                    return __fmaf_rn(-row.slope, __builtin_fabsf(__fadd_rn(to, -(float)(16 * (i >> 2) + (i & 3)))), __fmul_rn(x, f));
                });
            }
        }
        if (!whole) {
            const int lo = row.lo - at.first[p], hi = row.hi - at.first[p];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * kt + 4 * g + r;
                    t[p][kt][r] = j < lo || j >= hi ? -__builtin_inff() : __fmul_rn(t[p][kt][r], unit_of[p]);
                }
            unit_of[p] = 1.f;
        }
        float m = t[p][0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) m = fmaxf(m, t[p][i >> 2][i & 3]);
        most_of[p] = __fmul_rn(quad_max(m), unit_of[p]);
    }
    keys_done();
    float most = most_of[0];
#pragma unroll
    for (int p = 1; p < NP; ++p) most = fmaxf(most, most_of[p]);
    const bool sees = most != -__builtin_inff();
    const float base = sees ? most : 0.f;
    // weights times value scales are at most `unit`
    float unit = 0.f, times[NP];
    if constexpr (NP == 1) unit = at.v_scale[0], times[0] = WEIGHT_UNITS;
    else {
#pragma unroll
        for (int p = 0; p < NP; ++p) unit = fmaxf(unit, __fmul_rn(fast_exp2(__fadd_rn(most_of[p], -base)), at.v_scale[p]));
        // (finite whatever the scales: a page that the row does not see may have one that is far larger)
        const float per = unit > 0.f ? fminf(__fmul_rn(__builtin_amdgcn_rcpf(unit), WEIGHT_UNITS), 0x1p124f) : 0.f;
#pragma unroll
        for (int p = 0; p < NP; ++p) times[p] = fminf(__fmul_rn(at.v_scale[p], per), 0x1p126f);
    }
    // The exact product less the rounded maximum can be above 0, by 2^-24 of it. Up to 2^12 the weights' three digits have room for that;
    // scores beyond are rounded first.
    if (EXTRA == 0 && __any(__builtin_fabsf(base) > 0x1p12f)) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
#pragma unroll
            for (int i = 0; i < 16; ++i) t[p][i >> 2][i & 3] = __fmul_rn(t[p][i >> 2][i & 3], unit_of[p]);
            unit_of[p] = 1.f;
        }
    }
    float rest = 0.f;
    if constexpr (REST) {
        const float share = fast_exp2(__fadd_rn(EXTRA == 2 && KC == 1 ? __fadd_rn(most, away) : most, -s.m));
        const float put = __fmul_rn(__fmul_rn(share, 1.f / WEIGHT_UNITS), unit);
        rest = sees && put > finer.least ? put : 0.f;
        if (!__any(rest > 0.f)) return;
    }
    float sum = 0.f;
    v4i w[NP][3];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            unsigned u[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = fast_exp2(__fmaf_rn(t[p][kt][r], unit_of[p], -base));
                const float number = __fmaf_rn(e, times[p], 8388608.f + 32896.f);  // 2^23 + 0x8080: the mantissa is the rounded number
                if constexpr (!REST) {
                    sum = __fadd_rn(sum, e);
                    u[r] = __float_as_uint(number);
                } else {  // (the differences are exact, or to 24 bits of the weight itself)
                    float left = __fmul_rn(__fmaf_rn(e, times[p], -__fadd_rn(number, -(8388608.f + 32896.f))), 0x1p23f);
                    for (int n = 1; n < finer.level; ++n) left = __fmul_rn(__fadd_rn(left, -__builtin_rintf(left)), 0x1p23f);
                    u[r] = (unsigned)((int)__builtin_rintf(left) + 0x8080);
                }
            }
            int low, mid, high;
            split_digits(u, low, mid, high);
            w[p][2][kt] = low, w[p][1][kt] = mid, w[p][0][kt] = high;
        }
    if constexpr (EXTRA == 2 && KC == 1) most = __fadd_rn(most, away);
    if constexpr (REST) {
        const float per = __uint_as_float((unsigned)(127 - 23 * finer.level) << 23);
#pragma unroll
        for (int dt = 0; dt < 4 * KC; ++dt) {
            v4i a[3] = {};
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const v4i v = value(p, dt);
#pragma unroll
                for (int n = 0; n < 3; ++n) a[n] = mma(v, w[p][n], a[n]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s.o[dt][r] = __fmaf_rn(__fmul_rn(join_digits(a[0][r], a[1][r], a[2][r]), per), rest, s.o[dt][r]);
        }
        return;
    }
    const float m = fmaxf(s.m, most);
    const float keep = s.m == -__builtin_inff() ? 0.f : fast_exp2(__fadd_rn(s.m, -m));
    const float take = sees && (EXTRA != 2 || most != -__builtin_inff()) ? fast_exp2(__fadd_rn(most, -m)) : 0.f;
    s.second = __builtin_amdgcn_fmed3f(s.second, s.m, most);
    s.m = m;
    s.l = __fmaf_rn(s.l, keep, __fmul_rn(sum, take));
    const float put = __fmul_rn(__fmul_rn(take, 1.f / WEIGHT_UNITS), unit);
#pragma unroll
    for (int p = 0; p < NP; ++p) steps.scale = max(steps.scale, __float_as_uint(at.v_scale[p]));
    if (!__all(keep == 1.f)) {  // (a maximum seldom grows once a few pages are in)
        steps.raised |= 1ull << min(steps.now, 63);
#pragma unroll
        for (int dt = 0; dt < 4 * KC; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) s.o[dt][r] = __fmul_rn(s.o[dt][r], keep);
    }
#pragma unroll
    for (int dt = 0; dt < 4 * KC; ++dt) {
        v4i a[3] = {};
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const v4i v = value(p, dt);
#pragma unroll
            for (int n = 0; n < 3; ++n) a[n] = mma(v, w[p][n], a[n]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s.o[dt][r] = __fmaf_rn(join_digits(a[0][r], a[1][r], a[2][r]), put, s.o[dt][r]);
    }
    values_done();
}

// A sequence's pages as a wave walks them: their numbers come 64 at a time, one a lane.
struct PageWalk {
    const int32_t* table;
    int from, to, ids;
    __device__ int id(int pg) {  // pg: from, from + 1, ...
        if (((pg - from) & 63) == 0) ids = table[min(pg + (int)(threadIdx.x & 63), to - 1)];
        return __builtin_amdgcn_readlane(ids, (pg - from) & 63);
    }
};
// Pages pg .. pg + NP - 1, those behind the last and those that are none of the pool as pages whose tokens nobody sees, whatever is read
// in their place.
template <int NP>
__device__ __forceinline__ Pages<NP> pages_at(const KvView& c, int head, PageWalk& walk, int pg, const int8_t* (&kp)[NP], const int8_t* (&vp)[NP]) {
    Pages<NP> at;
    at.all = true;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int id = pg + n < walk.to ? walk.id(pg + n) : -1;
        const bool is = (unsigned)id < (unsigned)c.n_pages;
        const int page = is ? id : 0;
        kp[n] = c.k + c.at(page, head), vp[n] = c.v + c.at(page, head);
        const size_t sc = (size_t)page * c.heads + head;
        at.k_scale[n] = c.ks[sc], at.v_scale[n] = is ? c.vs[sc] : 0.f;
        at.first[n] = is ? (pg + n) * KV_BLOCK : 1 << 30;
        at.all = at.all && is;
    }
    return at;
}

template <int KC>
constexpr int kv_lds_bytes(bool staged, int waves) {
    const int join = waves * 16 * (64 * KC + 4) * 4 + waves * 16 * 2 * 4, stage = 2 * 8 * KC * 1024;
    return staged && stage > join ? stage : join;
}

// 64 rows a workgroup, one key head: a wave has a tile of 16 of them, or several waves share a tile's pages out between them and join
// what they have in LDS. A wave's next page is on its way into registers while it works on one. With STAGED and more than 32 rows the
// four waves read their pages, which are the same, from LDS, two at a time (see attend_pages), the next two on their way into registers: the
// faster way only where it leaves room for three workgroups a compute unit and there are as many, by 6 % for 65 to 128 dims (4096 rows on 14
// thousand tokens: 1.33 ms, 1.45 without, and 1.46 with two buffers in LDS and two workgroups). Without cap and slopes up to 64 dims leave
// room for four waves a SIMD if the compiler is told so (128 registers, else 130).
template <int KC, int EXTRA, bool STAGED, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, STAGED ? 3 : KC == 1 && EXTRA == 0 ? 4 : EXTRA < 2 ? 1 : KC == 1 ? 3 : KC <= 3 ? 2 : 1)
    kv_attend_kernel(AttendArgs a) {
    static_assert(!STAGED || WAVES == 4, "the staging is dealt to four waves");
    __shared__ __attribute__((aligned(16))) unsigned char lds[kv_lds_bytes<KC>(STAGED, WAVES)];
    typedef float JoinedRows[16][64 * KC + 4];
    JoinedRows* const joined = reinterpret_cast<JoinedRows*>(lds);
    typedef float JoinedSums[16][2];
    JoinedSums* const joined_ml = reinterpret_cast<JoinedSums*>(lds + sizeof(JoinedRows) * WAVES);
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4;
    const unsigned lane16 = (unsigned)lane * 16u;
    const int head = (int)(blockIdx.x % (unsigned)a.c.heads);
    const int tile = (int)(blockIdx.x / (unsigned)a.c.heads);
    const KvSeq s = kv_locate<64, false, true>(a.b.starts, a.b.lengths, a.b.n_seqs, a.b.n_tokens, a.group, tile);
    const int rows = s.count * a.group, last = ((rows + 63) >> 6) - 1;
    if (s.tile < 0 || s.tile > last) return;
    const int row0 = (last - s.tile) * 64;  // (a causal prompt's last rows have the most to read: they come first)
    const int tiles = (min(rows - row0, 64) + 15) >> 4;      // of 16 rows
    const int shares = tiles == 1 ? WAVES : tiles == 2 ? WAVES / 2 : WAVES / 4;  // waves that share a tile's pages
    const int mine = wave / shares, share = wave % shares;                      // (the last of three tiles have none: they join the barriers)
    const bool works = mine < tiles;
    const int r = row0 + mine * 16 + (lane & 15);
    const int row = min(r, rows - 1), token = row / a.group, q_head = head * a.group + row % a.group;
    const int p = s.first + token;
    const size_t out_row = (size_t)(s.begin + token) * a.q_heads + q_head;
    // positions that a row at p sees: [lo, hi)
    const int stored = min(s.length, a.b.max_pages * KV_BLOCK);
    const auto sees_to = [&](int p) { return p < 0 ? 0 : a.causal ? min(stored, p + 1) : stored; };
    const auto sees_from = [&](int p) { return a.window > 0 && p >= a.window ? p - a.window + 1 : 0; };
    RowView view;
    view.lo = sees_from(p), view.hi = sees_to(p), view.p = p, view.slope = 0.f;
    if constexpr (EXTRA == 2) {
        view.slope = __fmul_rn(a.slopes[q_head], LOG2E);
        if constexpr (KC == 1)
#pragma unroll
            for (int i = 0; i < 16; ++i) view.rise[i >> 2][i & 3] = __fmul_rn(view.slope, (float)(16 * (i >> 2) + 4 * g + (i & 3) - (KV_BLOCK - 1)));
    }
    const int first_p = __builtin_amdgcn_readlane(p, 0);
    Cap cap = a.cap;
    if constexpr (EXTRA != 0) {  // (held in registers: left alone the compiler loads them again for every page, and waits)
        asm volatile("" : "+s"(cap.cap));
#pragma unroll
        for (int n = 0; n < TANH_TERMS; ++n) asm volatile("" : "+s"(cap.half[n]));
    }
    // what the wave's rows see: rows are in the order of their tokens
    const int first_hi = __builtin_amdgcn_readlane(view.hi, 0), last_hi = __builtin_amdgcn_readlane(view.hi, 15);
    const int first_lo = __builtin_amdgcn_readlane(view.lo, 0), last_lo = __builtin_amdgcn_readlane(view.lo, 15);

    Running<KC> run;
    run.m = -__builtin_inff(), run.l = 0.f, run.second = -__builtin_inff();
#pragma unroll
    for (int dt = 0; dt < 4 * KC; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) run.o[dt][e] = 0.f;
    PageWalk walk;
    walk.table = a.b.pages + (size_t)s.index * a.b.max_pages;
    // pages [begin, end) of positions [lo, hi), the part-th of `parts` equal shares
    const auto deal = [&](int lo, int hi, int part, int parts) {
        const int page0 = lo / KV_BLOCK, pages = max((hi + KV_BLOCK - 1) / KV_BLOCK - page0, 0), each = (pages + parts - 1) / parts;
        walk.from = page0 + min(part * each, pages), walk.to = page0 + min((part + 1) * each, pages);
    };
    Queries<KC> q;
    float factor = 0.f;
    const auto load_rows = [&] {
        const bool whole_rows = a.c.dim % 4 == 0 && a.q_stride % 4 == 0 && ((size_t)a.q & 15) == 0;
        load_queries<KC>(q, a.q + (size_t)(s.begin + token) * a.q_stride + (size_t)q_head * a.c.dim, a.c.dim, whole_rows, a.scale < 0.f);
        factor = __fmul_rn(q.unit, __builtin_fabsf(a.scale));
    };
    const auto nothing = [] {};
    // Steps of NP pages, as they were taken, once more for the rows of which the rounding of the weights has left too little: whose largest element
    // is below ROUGH of the units, those of the step with the maximum and the root of the others' squares at the most. Mostly the first is what is
    // large, and only steps that raised a maximum are gone through; with the others too if they alone may be too much. At the end of the walk, since
    // only then is it known what o is: an ordinary row pays 20 to 40 instructions (the launch for one token on 520 takes 0.3 us more), and batches
    // whose rows all have such a token at their front 3 to 6 % (4096 rows on 14 thousand tokens: 1.35 -> 1.43 ms).
    Steps steps = {0, 0, 0};
    const auto finer = [&](auto pages) {
        constexpr int NP = decltype(pages)::value;
        const float many = __builtin_amdgcn_sqrtf((float)((walk.to - walk.from + NP - 1) / NP));
        const float others = __fmul_rn(__fmul_rn(fast_exp2(__fadd_rn(run.second, -run.m)), steps.unit()), many);
        float rough = ROUGH;
#pragma unroll 1
        for (int level = 1; level <= 3; ++level, rough *= 0x1p-23f) {
            float size = 0.f;
#pragma unroll
            for (int dt = 0; dt < 4 * KC; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) size = fmaxf(size, __builtin_fabsf(run.o[dt][e]));
            size = quad_max(size);
            const bool some = run.m != -__builtin_inff() && size < __fmul_rn(__fadd_rn(steps.unit(), others), rough);
            const bool all = size < __fmul_rn(others, rough);
            if (__builtin_expect(!__any(some), 1)) return;
            const Finer now = {some ? __fdiv_rn(size, __fmul_rn(many, rough)) : __builtin_inff(), level};
#pragma unroll 1
            for (int pg = walk.from, step = 0; pg < walk.to; pg += NP, ++step) {
                if (!steps.raises(step) && !__any(all)) continue;
                PageWalk one = {walk.table, pg, min(pg + NP, walk.to), 0};
                const int8_t *kp[NP], *vp[NP];
                const Pages<NP> at = pages_at<NP>(a.c, head, one, pg, kp, vp);
                const auto from = [&](const int8_t* page, int tile) { return *reinterpret_cast<const v4i*>(page + tile * 1024 + lane16); };
                attend_pages<KC, EXTRA, NP, true>(
                    run, q, [&](int n, int tile) { return from(kp[n], tile); }, [&](int n, int tile) { return from(vp[n], tile); }, nothing, nothing,
                    at, factor, cap, view, at.all && (pg + NP) * KV_BLOCK <= first_hi && pg * KV_BLOCK >= last_lo,
                    NP == 1 && (pg + 1) * KV_BLOCK <= first_p + 1, steps, now);
            }
        }
    };
    if (STAGED && shares == 1) {
        if constexpr (STAGED) {
            constexpr int NP = 2, TILES = NP * 8 * KC, MINE = TILES / 4;
            v4i* const buffer = reinterpret_cast<v4i*>(lds);  // [page][4 KC tiles of keys, as many of values][lane]
            const int p0 = s.first + row0 / a.group, p1 = s.first + (min(row0 + 64, rows) - 1) / a.group;
            deal(sees_from(p0), sees_to(p1), (int)blockIdx.y, a.splits);
            if (walk.from < walk.to) {
                load_rows();
                v4i mine_of[MINE];
                Pages<NP> at, next;
                const auto load = [&](int pg) {
                    const int8_t *kp[NP], *vp[NP];
                    next = pages_at<NP>(a.c, head, walk, pg, kp, vp);
#pragma unroll
                    for (int u = 0; u < MINE; ++u) {
                        const int j = wave * MINE + u, n = j / (8 * KC), of = j % (8 * KC);
                        const int8_t *const k = n ? kp[1] : kp[0], *const v = n ? vp[1] : vp[0];
                        mine_of[u] = *reinterpret_cast<const v4i*>((of < 4 * KC ? k + of * 1024 : v + (of - 4 * KC) * 1024) + lane16);
                    }
                };
                const auto put = [&] {
#pragma unroll
                    for (int u = 0; u < MINE; ++u) buffer[(wave * MINE + u) * 64 + lane] = mine_of[u];
                };
                load(walk.from);
                for (int pg = walk.from; pg < walk.to; pg += NP) {
                    at = next;
                    put();
                    if (pg + NP < walk.to) load(pg + NP);
                    // these pages are in LDS (loads from memory stay in flight)
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    if (works && pg * KV_BLOCK < last_hi && (pg + NP) * KV_BLOCK > first_lo) {
                        const bool whole = at.all && (pg + NP) * KV_BLOCK <= first_hi && pg * KV_BLOCK >= last_lo;
                        const v4i* const from = buffer + lane;
                        steps.now = (pg - walk.from) / NP;
                        attend_pages<KC, EXTRA, NP, false>(
                            run, q, [&](int n, int tile) { return from[(n * 8 * KC + tile) * 64]; },
                            [&](int n, int tile) { return from[(n * 8 * KC + 4 * KC + tile) * 64]; }, nothing, nothing, at, factor, cap, view, whole,
                            false, steps);
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // nobody reads them any more
                }
                finer(std::integral_constant<int, NP>{});
            }
        }
    } else if (works) {
        deal(first_lo, last_hi, (int)blockIdx.y * shares + share, a.splits * shares);
        if (walk.from < walk.to) {
            load_rows();
            v4i keys[4 * KC], values[4 * KC];
            const int8_t *kp[1], *vp[1];
            Pages<1> at = pages_at<1>(a.c, head, walk, walk.from, kp, vp);
            const auto load = [&](v4i (&to)[4 * KC], const int8_t* page) {
#pragma unroll
                for (int n = 0; n < 4 * KC; ++n) to[n] = *reinterpret_cast<const v4i*>(page + n * 1024 + lane16);
                __builtin_amdgcn_sched_barrier(0);  // (they are asked for here, not where they are used)
            };
            load(keys, kp[0]);
            load(values, vp[0]);
            const auto page = [&](int pg, const auto& keys_done, const auto& values_done) {
                const bool whole = at.all && (pg + 1) * KV_BLOCK <= first_hi && pg * KV_BLOCK >= last_lo;
                steps.now = pg - walk.from;
                attend_pages<KC, EXTRA, 1, false>(
                    run, q, [&](int, int tile) { return keys[tile]; }, [&](int, int tile) { return values[tile]; }, keys_done, values_done, at, factor,
                    cap, view, whole, (pg + 1) * KV_BLOCK <= first_p + 1, steps);
            };
            int pg = walk.from;
            for (; pg + 1 < walk.to; ++pg) {
                const Pages<1> next = pages_at<1>(a.c, head, walk, pg + 1, kp, vp);
                page(pg, [&] { load(keys, kp[0]); }, [&] { load(values, vp[0]); });
                at = next;
            }
            page(pg, nothing, nothing);
            finer(std::integral_constant<int, 1>{});
        }
    }
    run.l = quad_sum(run.l);
    if (shares > 1) {
        if (works) {
#pragma unroll
            for (int dt = 0; dt < 4 * KC; ++dt)
                *reinterpret_cast<float4*>(&joined[wave][lane & 15][dt * 16 + g * 4]) = {run.o[dt][0], run.o[dt][1], run.o[dt][2], run.o[dt][3]};
            if (g == 0) joined_ml[wave][lane & 15][0] = run.m, joined_ml[wave][lane & 15][1] = run.l;
        }
        __syncthreads();
        if (!works || share != 0) return;
        float m = run.m;
        for (int n = 1; n < shares; ++n) m = fmaxf(m, joined_ml[wave + n][lane & 15][0]);
        float keep = run.m == -__builtin_inff() ? 0.f : fast_exp2(__fadd_rn(run.m, -m));
        run.l = __fmul_rn(run.l, keep);
#pragma unroll
        for (int dt = 0; dt < 4 * KC; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) run.o[dt][e] = __fmul_rn(run.o[dt][e], keep);
        for (int n = 1; n < shares; ++n) {
            const float mn = joined_ml[wave + n][lane & 15][0];
            keep = mn == -__builtin_inff() ? 0.f : fast_exp2(__fadd_rn(mn, -m));
            run.l = __fmaf_rn(joined_ml[wave + n][lane & 15][1], keep, run.l);
#pragma unroll
            for (int dt = 0; dt < 4 * KC; ++dt) {
                const float4 f = *reinterpret_cast<const float4*>(&joined[wave + n][lane & 15][dt * 16 + g * 4]);
                run.o[dt][0] = __fmaf_rn(f.x, keep, run.o[dt][0]), run.o[dt][1] = __fmaf_rn(f.y, keep, run.o[dt][1]);
                run.o[dt][2] = __fmaf_rn(f.z, keep, run.o[dt][2]), run.o[dt][3] = __fmaf_rn(f.w, keep, run.o[dt][3]);
            }
        }
        run.m = m;
    }
    if (!works || r >= rows) return;
    float* to = a.out;
    size_t at = out_row;
    float by = run.l == 0.f ? 0.f : __fdiv_rn(1.f, run.l);  // (a row that sees nothing is 0)
    if (a.splits > 1) {
        at = (size_t)blockIdx.y * ((size_t)a.b.n_tokens * a.q_heads) + out_row;
        to = a.part_o;
        by = 1.f;
        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = {run.m, run.l};
        if (run.l == 0.f) return;  // (kv_join_kernel reads no sums of an empty share)
    }
    to += at * a.c.dim;
    const bool quads = a.c.dim % 4 == 0 && ((size_t)to & 15) == 0;
#pragma unroll
    for (int dt = 0; dt < 4 * KC; ++dt) {
        const int d = dt * 16 + g * 4;
        if (quads) {
            if (d < a.c.dim)
                *reinterpret_cast<float4*>(to + d) = {__fmul_rn(run.o[dt][0], by), __fmul_rn(run.o[dt][1], by), __fmul_rn(run.o[dt][2], by),
                                                      __fmul_rn(run.o[dt][3], by)};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < a.c.dim) to[d + e] = __fmul_rn(run.o[dt][e], by);
        }
    }
}

// The splits of a row joined, a row being a (token, query head): by a wave, or where they are many by the four of a workgroup, a quarter
// of the splits each, whose sums meet in LDS. A wave walks its splits eight at a time, so that their loads are in flight together. (One by
// one, by a single wave, 128 splits of 28 rows took 110 us; a workgroup for each of 12800 rows of two splits 25 us.)
template <int WAVES>
__global__ void __launch_bounds__(256) kv_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, float* __restrict__ out,
                                                      const int32_t* __restrict__ starts, int n_seqs, int n_rows, int q_heads, int dim, int splits) {
    __shared__ float sums[4][256];
    __shared__ float share_of[4][2];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int row = WAVES == 4 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave, share = WAVES == 4 ? wave : 0;
    const int token = row / q_heads;
    if (row >= n_rows || token < starts[0] || token >= starts[n_seqs]) return;  // rows of no sequence stay as they were
    const int each = (splits + WAVES - 1) / WAVES, from = min(share * each, splits), to = min(from + each, splits);
    // the wave's largest maximum; NaN weights have none: -infinity and a sum that is not 0
    float m = -__builtin_inff();
    for (int n = from + lane; n < to; n += 64) m = fmaxf(m, part_ml[2 * ((size_t)n * n_rows + row)]);
#pragma unroll
    for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int n0 = from; n0 < to; n0 += 64) {
        // a split for each lane: its weight
        float keep = 0.f, ln = 0.f;
        if (n0 + lane < to) {
            const float2 ml = *reinterpret_cast<const float2*>(part_ml + 2 * ((size_t)(n0 + lane) * n_rows + row));
            ln = ml.y;
            if (ln != 0.f) keep = ml.x == -__builtin_inff() ? 1.f : fast_exp2(__fadd_rn(ml.x, -m));
        }
        const int count = min(to - n0, 64);
        l = __fmaf_rn(ln, keep, l);
        for (int n = 0; n < count; n += 8) {
            float k[8], f[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                k[i] = n + i < count ? __shfl(keep, n + i) : 0.f;  // (of an empty split 0 too: its sums are not written)
                const float* const at = part_o + ((size_t)(n0 + min(n + i, count - 1)) * n_rows + row) * dim;
#pragma unroll
                for (int e = 0; e < 4; ++e) f[i][e] = n + i < count && lane + 64 * e < dim ? at[lane + 64 * e] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = k[i] != 0.f ? __fmaf_rn(f[i][e], k[i], o[e]) : o[e];
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) l = __fadd_rn(l, __shfl_xor(l, k));
    if constexpr (WAVES == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < dim) out[(size_t)row * dim + lane + 64 * e] = l == 0.f ? 0.f : __fdiv_rn(o[e], l);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave][lane + 64 * e] = o[e];
        if (lane == 0) share_of[wave][0] = m, share_of[wave][1] = l;
        __syncthreads();
        m = fmaxf(fmaxf(share_of[0][0], share_of[1][0]), fmaxf(share_of[2][0], share_of[3][0]));
        float total = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float lw = share_of[w][1], mw = share_of[w][0];
            const float keep = lw == 0.f ? 0.f : mw == -__builtin_inff() ? 1.f : fast_exp2(__fadd_rn(mw, -m));
            total = __fmaf_rn(lw, keep, total);
            sum = __fmaf_rn(sums[w][threadIdx.x], keep, sum);
        }
        if ((int)threadIdx.x < dim) out[(size_t)row * dim + threadIdx.x] = total == 0.f ? 0.f : __fdiv_rn(sum, total);
    }
}

// How a batch is launched, by the tiles that its rows fill if they are spread evenly: the sizes of its sequences are on the GPU.
//   staged  from three workgroups a compute unit on, more being there to follow (extra: cap or slopes, which take its registers)
//   waves   of a workgroup: four where the tiles give every compute unit more than one, as many as their loads need to fill its memory pipe
//           (and over 192 dims, where eight have too few registers), else eight. One token on 520 tokens, 4 heads of 64: 6.9 us with
//           four, 6.2 with eight; 16 x 64 rows on 4000 tokens, 8 heads of 128: 86 and 70
//   splits  shares that the pages of a tile are cut into, each a workgroup's: as many as give the compute units eight waves at the most, but
//           four pages to a wave at least: joining the shares takes another launch, as long as four pages do. 64 rows on 16 thousand tokens:
//           240 us in one share, 53 in eight
KvPlan kv_attend_plan(int n_tokens, int n_seqs, int group, int heads, int chunks, bool extra, int max_pages) {
    const size_t rows = (size_t)n_tokens * group, even = (rows + 63) / 64, seqs = (size_t)n_seqs;
    const size_t have = (even > seqs ? even : seqs) * heads;
    KvPlan p;
    p.staged = chunks == 2 && !extra && have >= 1024 && rows > 32 * seqs;
    p.waves = have > 256 || chunks > 3 ? 4 : 8;
    const int tiles = rows <= 16 * seqs ? 1 : rows <= 32 * seqs ? 2 : 4;  // of 16 rows, which the waves of a workgroup are dealt to
    const size_t fill = 2048 / p.waves / have, want = have > 256 || fill < 1 ? 1 : fill, most = (size_t)max_pages / (4 * (p.waves / tiles));
    p.splits = (int)(want < most ? want : most < 1 ? 1 : most);
    return p;
}
int kv_attend_tiles(int n_tokens, int n_seqs, int group) { return (int)((size_t)n_tokens * group / 64) + n_seqs; }

template <int KC, int WAVES>
static void launch_attend(const AttendArgs& a, dim3 grid, hipStream_t stream) {
    if (a.slopes) launch(kv_attend_kernel<KC, 2, false, WAVES>, grid, dim3(64 * WAVES), 0, stream, a);
    else if (a.cap.cap != 0.f) launch(kv_attend_kernel<KC, 1, false, WAVES>, grid, dim3(64 * WAVES), 0, stream, a);
    else launch(kv_attend_kernel<KC, 0, false, WAVES>, grid, dim3(64 * WAVES), 0, stream, a);
}
template <int KC>
static void launch_attend(const AttendArgs& a, const KvPlan& p, dim3 grid, hipStream_t stream) {
    if constexpr (KC == 2) {
        if (p.staged) return launch(kv_attend_kernel<2, 0, true, 4>, grid, dim3(256), 0, stream, a);
    }
    if constexpr (KC <= 3) {
        if (p.waves == 8) return launch_attend<KC, 8>(a, grid, stream);
    }
    launch_attend<KC, 4>(a, grid, stream);
}

hipError_t run_kv_attend(const KvView& c, const KvBatch& b, const float* q, size_t q_stride, float* out, int q_heads, float scale, float cap,
                         const float* slopes, int causal, int window, const KvPlan& plan, void* workspace, hipStream_t stream) {
    const int splits = plan.splits;
    AttendArgs a;
    a.c = c, a.b = b, a.q = q, a.q_stride = q_stride, a.out = out, a.q_heads = q_heads, a.group = q_heads / c.heads;
    a.scale = cap != 0.f ? scale / cap : scale * LOG2E;
    a.cap.cap = cap * LOG2E;
    for (int n = 0; n < TANH_TERMS; ++n) a.cap.half[n] = (float)((double)a.cap.cap * TANH_TERM[n]);
    a.slopes = slopes, a.causal = causal, a.window = window;
    a.tiles = kv_attend_tiles(b.n_tokens, b.n_seqs, a.group), a.splits = splits;
    const size_t rows = (size_t)b.n_tokens * q_heads;
    a.part_ml = (float*)workspace;
    a.part_o = a.part_ml + (splits > 1 ? (2 * rows * splits + 3) / 4 * 4 : 0);
    const dim3 grid((unsigned)a.tiles * (unsigned)c.heads, (unsigned)splits);
    switch (c.chunks) {
    case 1: launch_attend<1>(a, plan, grid, stream); break;
    case 2: launch_attend<2>(a, plan, grid, stream); break;
    case 3: launch_attend<3>(a, plan, grid, stream); break;
    default: launch_attend<4>(a, plan, grid, stream); break;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || splits == 1) return e;
    const auto join = [&](auto kernel, size_t groups) {
        launch(kernel, dim3((unsigned)groups), dim3(256), 0, stream, (const float*)a.part_o, (const float*)a.part_ml, out, b.starts, b.n_seqs, (int)rows,
               q_heads, c.dim, splits);
    };
    if (splits > 16) join(kv_join_kernel<4>, rows);
    else join(kv_join_kernel<1>, (rows + 3) / 4);
    return hipGetLastError();
}

}  // namespace ohip
