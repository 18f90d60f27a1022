// Int8 products grouped by expert: y = act(codes(x) . W[e] * (x_scale * w_scale[e]) + bias[e]), rows sorted by expert.
//
// Rows come as floats. A first launch finds each row's scale, largest size / 127, and rounds the row to codes (exactly, code_of); the
// second multiplies on the int8 matrix cores. The sums are exact in 32 bits, so it does not matter in what order or by how many waves
// they are formed.
#include "kv_common.hpp"
#include "linear.hpp"

namespace ohip {

typedef ohip_v4i v4i;

struct LinearCodes {
    float* scale;   // [x_rows]
    int8_t* codes;  // [x_rows][whole pairs of steps]
};
static LinearCodes linear_codes(const LinearView& w, int x_rows, void* workspace) {
    LinearCodes c;
    c.scale = (float*)workspace;
    c.codes = (int8_t*)workspace + ((size_t)x_rows * 4 + 255) / 256 * 256;
    return c;
}
// bytes of a row of codes: whole pairs of steps, zeros behind the last input
__host__ __device__ inline size_t linear_row_bytes(int steps) { return (size_t)(steps + 1) / 2 * 128; }
size_t linear_workspace_bytes(const LinearView& w, int x_rows) { return ((size_t)x_rows * 4 + 255) / 256 * 256 + (size_t)x_rows * linear_row_bytes(w.steps); }

// Weights into tiles of 16 outputs x 64 inputs, in the order of the matrix instruction's lanes: a thread a piece, 16 inputs of an output
// (zeros behind the last of either).
__global__ void __launch_bounds__(256) linear_pack_kernel(const int8_t* __restrict__ weight, int8_t* __restrict__ tiles, size_t pieces, int out, int in,
                                                          int halves, int half_tiles, int steps) {
    for (size_t piece = (size_t)blockIdx.x * 256 + threadIdx.x; piece < pieces; piece += (size_t)gridDim.x * 256) {
        const int lane = (int)(piece & 63);
        const size_t tile = (piece >> 6) / (unsigned)steps;  // of all experts, the halves in turn
        const int step = (int)((piece >> 6) % (unsigned)steps), half = (int)(tile % (unsigned)halves);
        const size_t pair = tile / (unsigned)halves, expert = pair / (unsigned)half_tiles;
        const int n = (int)(pair % (unsigned)half_tiles) * 16 + (lane & 15), k = step * 64 + (lane >> 4) * 16;
        int8_t v[16] __attribute__((aligned(16))) = {};
        if (n < out) {
            const int8_t* const from = weight + ((expert * halves + half) * (size_t)out + n) * in;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (k + i < in) v[i] = from[k + i];
        }
        *reinterpret_cast<v4i*>(tiles + piece * 16) = *reinterpret_cast<const v4i*>(v);
    }
}
hipError_t run_linear_pack(const int8_t* weight, int8_t* tiles, int experts, int out, int in, int halves) {
    const int half_tiles = (out + 15) / 16, steps = (in + 63) / 64;
    const size_t pieces = (size_t)experts * halves * half_tiles * steps * 64;
    launch(linear_pack_kernel, dim3((unsigned)std::min<size_t>((pieces + 255) / 256, 65536)), dim3(256), 0, nullptr, weight, tiles, pieces, out, in, halves, half_tiles, steps);
    return hipGetLastError();
}

// Four inputs of a row from d on; those behind its last are 0.
__device__ __forceinline__ float4 row_quad(const float* __restrict__ row, int d, int in, bool quads) {
    float4 f = {0.f, 0.f, 0.f, 0.f};
    if (quads) {
        if (d < in) f = *reinterpret_cast<const float4*>(row + d);
    } else {
        if (d < in) f.x = row[d];
        if (d + 1 < in) f.y = row[d + 1];
        if (d + 2 < in) f.z = row[d + 2];
        if (d + 3 < in) f.w = row[d + 3];
    }
    return f;
}
__device__ __forceinline__ float most_of_quad(const float4& f) {
    const float v[4] = {f.x, f.y, f.z, f.w};
    return largest_size(v);
}

// A workgroup a row: its largest size, then its codes. 4096 inputs stay in registers, what is behind them is read again.
__global__ void __launch_bounds__(256) linear_codes_kernel(const float* __restrict__ x, size_t stride, int in, int padded, float* __restrict__ scale,
                                                           int8_t* __restrict__ codes) {
    constexpr int KEPT = 4;
    __shared__ float most_of[4];
    const int tid = (int)threadIdx.x;
    const float* const row = x + (size_t)blockIdx.x * stride;
    const bool quads = in % 4 == 0 && stride % 4 == 0 && ((size_t)x & 15) == 0;
    float4 kept[KEPT];
#pragma unroll
    for (int u = 0; u < KEPT; ++u) kept[u] = row_quad(row, 4 * tid + 1024 * u, in, quads);
    float most = largest_size(reinterpret_cast<const float(&)[4 * KEPT]>(kept));
    for (int d = 4 * tid + 1024 * KEPT; d < in; d += 1024) most = fmaxf(most, most_of_quad(row_quad(row, d, in, quads)));
#pragma unroll
    for (int m = 32; m; m >>= 1) most = fmaxf(most, __shfl_xor(most, m));
    if ((tid & 63) == 0) most_of[tid >> 6] = most;
    __syncthreads();
    const float s = scale_of(fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3])));
    const Coder coder(s);
    if (tid == 0) scale[blockIdx.x] = s;
    int* const to = reinterpret_cast<int*>(codes + (size_t)blockIdx.x * padded);
    bool doubtful = false;
#pragma unroll
    for (int u = 0; u < KEPT; ++u)
        if (4 * tid + 1024 * u < padded) to[tid + 256 * u] = coder.word(kept[u].x, kept[u].y, kept[u].z, kept[u].w, doubtful);
    for (int d = 4 * tid + 1024 * KEPT; d < padded; d += 1024) {
        const float4 f = row_quad(row, d, in, quads);
        to[d >> 2] = coder.word(f.x, f.y, f.z, f.w, doubtful);
    }
    if (doubtful) {
#pragma unroll 1
        for (int d = 4 * tid; d < padded; d += 1024) {
            const float4 f = row_quad(row, d, in, quads);
            to[d >> 2] = coder.exact_word(f.x, f.y, f.z, f.w);
        }
    }
}

struct LinearArgs {
    LinearView w;
    const float* scale;
    const int8_t* codes;
    const int32_t *index, *starts;
    int x_rows, rows;
    float* y;
    bool streams;
};

// Expert and rows of a tile of UNIT rows: [begin, end), empty where the tile is behind its expert's rows.
struct LinearTile {
    int expert, begin, end;
    int all;  // tiles of all experts (-1: not counted)
};
template <int UNIT>
__device__ __forceinline__ LinearTile linear_tile(const LinearArgs& a, int tile) {
    LinearTile t;
    if (!a.starts) {
        t.expert = 0, t.begin = min(tile * UNIT, a.rows), t.end = min(t.begin + UNIT, a.rows), t.all = (a.rows + UNIT - 1) / UNIT;
        return t;
    }
    const KvSeq s = kv_locate<UNIT, false, false>(a.starts, nullptr, a.w.experts, a.rows, 1, tile);
    t.expert = s.index, t.all = s.all;
    const int to = s.begin + s.count;
    t.begin = s.tile < 0 ? to : min(s.begin + s.tile * UNIT, to);
    t.end = min(t.begin + UNIT, to);
    return t;
}
static int linear_row_tiles(const LinearView& w, const LinearRows& r, int unit) {
    return r.starts ? r.rows / unit + w.experts : (int)(((size_t)r.rows + unit - 1) / unit);
}

// Row of x behind a sorted row (an index outside of x: -1).
__device__ __forceinline__ int linear_source(const LinearArgs& a, int row) {
    const int i = a.index ? a.index[row] : row;
    return (unsigned)i < (unsigned)a.x_rows ? i : -1;
}

// What the epilogue needs of four consecutive outputs: a lane's share of an output tile.
struct LinearOut {
    float4 scale, bias;
};
__device__ __forceinline__ LinearOut linear_out(const LinearArgs& a, int expert, int tile) {
    const size_t at = ((size_t)expert * a.w.tiles + tile) * 16 + ((threadIdx.x >> 4) & 3) * 4;
    LinearOut o;
    o.scale = *reinterpret_cast<const float4*>(a.w.scale + at);
    o.bias = {0.f, 0.f, 0.f, 0.f};
    if (a.w.bias) o.bias = *reinterpret_cast<const float4*>(a.w.bias + at);
    return o;
}
__device__ __forceinline__ float4 linear_value(const v4i& acc, float xs, const LinearOut& o) {
    return {__fmaf_rn((float)acc[0], __fmul_rn(xs, o.scale.x), o.bias.x), __fmaf_rn((float)acc[1], __fmul_rn(xs, o.scale.y), o.bias.y),
            __fmaf_rn((float)acc[2], __fmul_rn(xs, o.scale.z), o.bias.z), __fmaf_rn((float)acc[3], __fmul_rn(xs, o.scale.w), o.bias.w)};
}
// What becomes of a result: an instance each, as 128 results of a lane with a choice in front of each were 24 thousand instructions, and a
// third of the time of a launch.
enum { LINEAR_PLAIN, LINEAR_CLAMP, LINEAR_LEAKY, LINEAR_SIGMOID, LINEAR_MISH, LINEAR_GATED };
static int linear_end(const LinearView& w) {
    switch (w.gated ? -1 : w.act) {
    case -1: return LINEAR_GATED;
    case 1:
    case 3: return LINEAR_CLAMP;
    case 2: return LINEAR_LEAKY;
    case 4: return LINEAR_SIGMOID;
    case 5: return LINEAR_MISH;
    default: return LINEAR_PLAIN;
    }
}
template <int END>
__device__ __forceinline__ float linear_act(float v, float up, float p0) {
    if constexpr (END == LINEAR_CLAMP) return fminf(fmaxf(v, 0.f), p0);  // (p0: 6 or infinity)
    if constexpr (END == LINEAR_LEAKY) return activate(v, 2, p0);
    if constexpr (END == LINEAR_SIGMOID) return activate(v, 4, p0);
    if constexpr (END == LINEAR_MISH) return activate(v, 5, p0);
    if constexpr (END == LINEAR_GATED) return __fmul_rn(__fdiv_rn(v, __fadd_rn(1.f, __expf(-v))), up);
    return v;
}
typedef float v4f __attribute__((ext_vector_type(4)));
// Four consecutive outputs of one row, `column` the first. Results beyond what the L2s hold (a.streams) are not kept there.
template <int END>
__device__ __forceinline__ void linear_store(const LinearArgs& a, int row, float xs, int n_tile, const v4i& acc, const v4i& acc_up, const LinearOut& o,
                                             const LinearOut& o_up, bool quads) {
    const float4 v = linear_value(acc, xs, o);
    float4 u = {0.f, 0.f, 0.f, 0.f};
    if constexpr (END == LINEAR_GATED) u = linear_value(acc_up, xs, o_up);
    const v4f r = {linear_act<END>(v.x, u.x, a.w.act_p0), linear_act<END>(v.y, u.y, a.w.act_p0), linear_act<END>(v.z, u.z, a.w.act_p0),
                   linear_act<END>(v.w, u.w, a.w.act_p0)};
    const int column = n_tile * 16 + (int)((threadIdx.x >> 4) & 3) * 4;
    float* const to = a.y + (size_t)row * a.w.out + column;
    if (quads) {
        if (column >= a.w.out) return;
        if (a.streams) __builtin_nontemporal_store(r, reinterpret_cast<v4f*>(to));
        else *reinterpret_cast<v4f*>(to) = r;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (column + e < a.w.out) to[e] = r[e];
    }
}
__device__ __forceinline__ bool linear_quads(const LinearArgs& a) { return a.w.out % 4 == 0 && ((size_t)a.y & 15) == 0; }

// 16 outputs (gated: 16 of either half) x 16 rows a workgroup, the inputs dealt to its W waves, whose sums meet in LDS. Both operands
// come straight from memory in lane order, several steps of them asked for before the first is used; this is the launch for few rows,
// where reading the weights is the work. It reads them once for every 16 rows: 64 rows of 4096 x 4096 take 15.9 us with their codes, 32 11.0.
template <int END, int W>
__global__ void __launch_bounds__(64 * W) linear_few_kernel(LinearArgs a) {
    constexpr int G = END == LINEAR_GATED ? 2 : 1, AHEAD = 4;
    __shared__ v4i sums[W][G][64];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const unsigned n_tiles = (unsigned)a.w.tiles / G;
    const int n_tile = (int)(blockIdx.x % n_tiles);
    const LinearTile t = linear_tile<16>(a, (int)(blockIdx.x / n_tiles));
    if (t.begin >= t.end) return;
    const int steps = a.w.steps;
    const int8_t* const w = a.w.w + ((size_t)t.expert * a.w.tiles + (size_t)n_tile * G) * steps * 1024;
    const unsigned lane16 = (unsigned)lane * 16u;
    const int row = t.begin + (lane & 15), src = linear_source(a, min(row, t.end - 1));
    const int8_t* const x = a.codes + (size_t)max(src, 0) * linear_row_bytes(steps) + (lane >> 4) * 16;
    v4i acc[G] = {};
    const int each = (steps + W - 1) / W, to = min((wave + 1) * each, steps);
    for (int s = wave * each; s < to; s += AHEAD) {
        v4i k[AHEAD][G], b[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int at = min(s + u, to - 1);
#pragma unroll
            for (int h = 0; h < G; ++h) k[u][h] = *reinterpret_cast<const v4i*>(w + ((size_t)h * steps + at) * 1024 + lane16);
            b[u] = *reinterpret_cast<const v4i*>(x + (size_t)at * 64);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (s + u >= to) break;
#pragma unroll
            for (int h = 0; h < G; ++h) acc[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[u][h], b[u], acc[h], 0, 0, 0);
        }
    }
#pragma unroll
    for (int h = 0; h < G; ++h) sums[wave][h][lane] = acc[h];
    __syncthreads();
    if (wave != 0 || row >= t.end) return;
    v4i sum[2] = {};
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
        for (int n = 0; n < W; ++n) sum[h] += sums[n][h][lane];
    const LinearOut o = linear_out(a, t.expert, n_tile * G), o_up = linear_out(a, t.expert, n_tile * G + G - 1);
    linear_store<END>(a, row, src < 0 ? 0.f : a.scale[src], n_tile, sum[0], sum[1], o, o_up, linear_quads(a));
}

// The same launch with the rows' codes found by every workgroup for itself, in LDS, while its first weights are on their way: for the
// row or two of a decoding step a launch in front of it takes as long as the product (one row of 2048 x 2048: 2.7 and 3.4 us). A row has
// W / (rows, rounded up to a power of two) waves, or a wave has several rows. 16-byte pieces of a row lie at their index xor (row / 2) % 8,
// so that the 16 rows of an operand spread over the banks.
template <int END, int W>
__global__ void __launch_bounds__(64 * W) linear_rows_kernel(LinearArgs a, const float* __restrict__ x, size_t x_stride) {
    constexpr int G = END == LINEAR_GATED ? 2 : 1, AHEAD = 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // codes [row][pieces], then the waves' sums
    __shared__ float most_of[16][W];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const unsigned n_tiles = (unsigned)a.w.tiles / G;
    const int n_tile = (int)(blockIdx.x % n_tiles);
    const LinearTile t = linear_tile<16>(a, (int)(blockIdx.x / n_tiles));
    const int count = t.end - t.begin;
    if (count <= 0) return;
    const int steps = a.w.steps, in = a.w.in;
    const int8_t* const w = a.w.w + ((size_t)t.expert * a.w.tiles + (size_t)n_tile * G) * steps * 1024;
    const unsigned lane16 = (unsigned)lane * 16u;
    const int each = (steps + W - 1) / W, from = wave * each, to = min(from + each, steps);
    v4i k[AHEAD][G];
    const auto load_w = [&](int s) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int h = 0; h < G; ++h) k[u][h] = *reinterpret_cast<const v4i*>(w + ((size_t)h * steps + min(s + u, steps - 1)) * 1024 + lane16);
    };
    load_w(min(from, steps - 1));
    // waves to a row, and the part of the rows' quads that a wave has
    const int shares = count >= W ? 1 : (count <= 1 ? W : W >> (32 - __clz(count - 1))), share = wave % shares, first = wave / shares, apart = W / shares;
    const int row_bytes = (int)linear_row_bytes(steps), quads_each = (row_bytes / 4 + shares - 1) / shares;
    const int q0 = share * quads_each, q1 = min(q0 + quads_each, row_bytes / 4);
    const bool quads = in % 4 == 0 && x_stride % 4 == 0 && ((size_t)x & 15) == 0;
    for (int r = first; r < count; r += apart) {
        const int src = linear_source(a, t.begin + r);
        const float* const row = x + (size_t)max(src, 0) * x_stride;
        float most = 0.f;
        for (int q = q0 + lane; q < q1; q += 64) most = fmaxf(most, most_of_quad(row_quad(row, 4 * q, in, quads)));
#pragma unroll
        for (int m = 32; m; m >>= 1) most = fmaxf(most, __shfl_xor(most, m));
        if (lane == 0) most_of[r][share] = src < 0 ? 0.f : most;
    }
    __syncthreads();
    const auto scale_of_row = [&](int r) {
        float most = most_of[r][0];
        for (int n = 1; n < shares; ++n) most = fmaxf(most, most_of[r][n]);
        return scale_of(most);
    };
    for (int r = first; r < count; r += apart) {
        const int src = linear_source(a, t.begin + r);
        const float* const row = x + (size_t)max(src, 0) * x_stride;
        const Coder coder(scale_of_row(r));
        for (int q = q0 + lane; q < q1; q += 64) {
            const int piece = (q >> 2) ^ ((r >> 1) & 7);
            const float4 f = row_quad(row, 4 * q, in, quads);
            bool doubtful = false;
            int code = coder.word(f.x, f.y, f.z, f.w, doubtful);
            if (doubtful) code = coder.exact_word(f.x, f.y, f.z, f.w);
            *reinterpret_cast<int*>(lds + r * row_bytes + piece * 16 + (q & 3) * 4) = code;
        }
    }
    __syncthreads();
    const int mine = min(lane & 15, count - 1);
    v4i acc[G] = {};
    for (int s = from; s < to; s += AHEAD) {
        if (s > from) load_w(s);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (s + u >= to) break;
            const int piece = ((s + u) * 4 + (lane >> 4)) ^ ((mine >> 1) & 7);
            const v4i b = *reinterpret_cast<const v4i*>(lds + mine * row_bytes + piece * 16);
#pragma unroll
            for (int h = 0; h < G; ++h) acc[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[u][h], b, acc[h], 0, 0, 0);
        }
    }
    __syncthreads();
    v4i* const sums = reinterpret_cast<v4i*>(lds);
#pragma unroll
    for (int h = 0; h < G; ++h) sums[(wave * G + h) * 64 + lane] = acc[h];
    __syncthreads();
    const int row = t.begin + (lane & 15);
    if (wave != 0 || row >= t.end) return;
    v4i sum[2] = {};
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
        for (int n = 0; n < W; ++n) sum[h] += sums[(n * G + h) * 64 + lane];
    const LinearOut o = linear_out(a, t.expert, n_tile * G), o_up = linear_out(a, t.expert, n_tile * G + G - 1);
    linear_store<END>(a, row, scale_of_row(mine), n_tile, sum[0], sum[1], o, o_up, linear_quads(a));
}

// 64 NT outputs x 16 RT rows a workgroup, 16 NT outputs a wave: the launch for many rows. A wave loads its weights, which no other
// wave of the workgroup reads, straight into registers, a stage of 128 inputs ahead; the rows' codes, which all four waves read, go
// through LDS, in lane order too (a 16-byte piece of a row is a lane's). A stage is 8 NT RT matrix instructions a wave against 2 RT KB
// from LDS and 2 NT KB from memory: with 4 and 8 that is 64 and 32 bytes a cycle of a compute unit's 128 and 64.
template <int NT, int RT>
struct LinearRing {
    v4i rows[3][RT][2][64];
};
template <int NT, int RT, int END>
__device__ __forceinline__ void linear_many(const LinearArgs& a, const LinearTile& t, int first_tile, void* lds) {
    constexpr int MINE = RT / 4;  // tiles of 16 rows that a wave brings in
    auto& rows = reinterpret_cast<LinearRing<NT, RT>*>(lds)->rows;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int tile0 = first_tile + wave * NT, steps = a.w.steps;
    const size_t row_bytes = linear_row_bytes(steps);
    const int8_t* w[NT];  // (the same for every lane: the lane's share is a 32-bit offset to it)
#pragma unroll
    for (int n = 0; n < NT; ++n) w[n] = a.w.w + ((size_t)t.expert * a.w.tiles + min(tile0 + n, a.w.tiles - 1)) * steps * 1024;
    const unsigned lane16 = (unsigned)lane * 16u;
    const int8_t* x[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int src = linear_source(a, min(t.begin + (wave * MINE + i) * 16 + (lane & 15), t.end - 1));
        x[i] = a.codes + (size_t)max(src, 0) * row_bytes + (lane >> 4) * 16;
    }
    // (steps go in twos: an odd count ends on a step of zeros of the rows)
    const int even = (steps + 1) & ~1;
    const auto load_w = [&](v4i (&to)[NT], int s) {
#pragma unroll
        for (int n = 0; n < NT; ++n) to[n] = *reinterpret_cast<const v4i*>(w[n] + (size_t)min(s, steps - 1) * 1024 + lane16);
    };
    v4i xr[MINE][2];
    const auto load_x = [&](int s) {
#pragma unroll
        for (int i = 0; i < MINE; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) xr[i][h] = *reinterpret_cast<const v4i*>(x[i] + (size_t)min(s, even - 2) * 64 + h * 64);
    };
    const auto put_x = [&](int slot) {
#pragma unroll
        for (int i = 0; i < MINE; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) rows[slot][wave * MINE + i][h][lane] = xr[i][h];
    };
    v4i acc[NT][RT] = {};
    v4i wr[4][NT];
    load_x(0);
    put_x(0);
    load_x(2);
#pragma unroll
    for (int s = 0; s < 4; ++s) load_w(wr[s], s);
    put_x(1);
    load_x(4);
    int slot = 0;
    // A stage: two steps. Weights are asked for four steps before their use, rows two stages before it, one before they go to LDS. No
    // branch in the loop: behind one the compiler waits for every load in flight.
    const auto stage = [&](auto parity, int s) {
        constexpr int P = decltype(parity)::value;
        // this stage's rows are in LDS, and nobody reads the slot before it any more (loads from memory stay in flight)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const v4i* const from = &rows[slot][0][0][lane];
        v4i b[3];
        b[0] = from[0], b[1] = from[128];
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i) {  // (row tile, step): a tile is read from LDS two tiles before its products
            const int h = i / RT, r = i % RT;
            if (i + 2 < 2 * RT) b[(i + 2) % 3] = from[((i + 2) % RT * 2 + (i + 2) / RT) * 64];
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wr[2 * P + h][n], b[i % 3], acc[n][r], 0, 0, 0);
            if (r == RT - 1) load_w(wr[2 * P + h], s + h + 4);
            if (i == RT - 1) {
                put_x(slot == 0 ? 2 : slot - 1);
                load_x(s + 6);
            }
            __builtin_amdgcn_sched_barrier(0);  // (left alone the compiler reads a tile right in front of its products)
        }
        slot = slot == 2 ? 0 : slot + 1;
    };
    int s = 0;
    for (; s + 4 <= even; s += 4) {
        stage(std::integral_constant<int, 0>{}, s);
        stage(std::integral_constant<int, 1>{}, s + 2);
    }
    if (s < even) stage(std::integral_constant<int, 0>{}, s);
    constexpr int G = END == LINEAR_GATED ? 2 : 1;
    float xs[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int src = linear_source(a, min(t.begin + r * 16 + (lane & 15), t.end - 1));
        xs[r] = src < 0 ? 0.f : a.scale[src];
    }
    const auto finish = [&](bool quads) {
        LinearOut o[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n] = linear_out(a, t.expert, min(tile0 + n, a.w.tiles - 1));
        // (the pieces of a row one behind the other: stores that pass the caches fill lines sooner. 8192 rows of 4096 x 4000 172.6 -> 170.0 us)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = t.begin + r * 16 + (lane & 15);
            if (row >= t.end) continue;
#pragma unroll
            for (int n = 0; n < NT; n += G)
                if (tile0 + n < a.w.tiles) linear_store<END>(a, row, xs[r], (tile0 + n) / G, acc[n][r], acc[n + G - 1][r], o[n], o[n + G - 1], quads);
        }
    };
    if (linear_quads(a)) finish(true);
    else finish(false);
}

// Two workgroups of 64 x 128 results a wave fill a compute unit. Where a grid of them is a few more than whole rounds, those few are cut in
// four each: one of them by itself takes 1.55 us a stage, a quarter 0.62. 4096 x 4096 with codes: 512 workgroups 85 us, 544: 93, 608: 107,
// 1056: 175. (Uncut, when these took 94, 99, 109 and 174: 544 113, 608 114, 640 115, 1056 189; and 640 cut 119. More than 64 experts: their
// tiles are not counted, and not cut.)
constexpr int LINEAR_PLACES = 512, LINEAR_CUT = 96;
template <int NT, int RT, int END>
__global__ void __launch_bounds__(256, 2) linear_many_kernel(LinearArgs a) {
    __shared__ LinearRing<NT, RT> lds;
    const int n_blocks = (a.w.tiles + 4 * NT - 1) / (4 * NT), group = (int)blockIdx.x;
    LinearTile t = linear_tile<16 * RT>(a, group / n_blocks);
    if constexpr (RT == 8) {
        const int all = t.all * n_blocks, over = all % LINEAR_PLACES;
        if (all >= LINEAR_PLACES && over <= LINEAR_CUT && group >= all - over) {
            const int part = group - (all - over), cut = all - over + (part >> 2);
            if (cut >= all) return;
            t = linear_tile<16 * RT>(a, cut / n_blocks);
            t.begin = min(t.begin + (part & 2) * 32, t.end);
            t.end = min(t.begin + 64, t.end);
            if (t.begin < t.end) linear_many<NT / 2, RT / 2, END>(a, t, (cut % n_blocks * 2 + (part & 1)) * 2 * NT, &lds);
            return;
        }
    }
    if (t.begin < t.end) linear_many<NT, RT, END>(a, t, group % n_blocks * 4 * NT, &lds);
}

#define OHIP_LINEAR_END(CALL)                                  \
    switch (linear_end(a.w)) {                                 \
    case LINEAR_GATED: CALL(LINEAR_GATED); break;              \
    case LINEAR_CLAMP: CALL(LINEAR_CLAMP); break;              \
    case LINEAR_LEAKY: CALL(LINEAR_LEAKY); break;              \
    case LINEAR_SIGMOID: CALL(LINEAR_SIGMOID); break;          \
    case LINEAR_MISH: CALL(LINEAR_MISH); break;                \
    default: CALL(LINEAR_PLAIN); break;                        \
    }
static size_t few_groups(const LinearView& w, const LinearRows& r) { return (size_t)(w.tiles / (w.gated ? 2 : 1)) * linear_row_tiles(w, r, 16); }
static size_t many_groups(const LinearView& w, const LinearRows& r, int nt, int rt) {
    const size_t n = (size_t)((w.tiles + 4 * nt - 1) / (4 * nt)) * linear_row_tiles(w, r, 16 * rt);
    return rt == 8 && n >= LINEAR_PLACES ? n + 3 * LINEAR_CUT : n;  // (with the quarters of those that are cut, however many the experts' rows make)
}
size_t linear_groups(const LinearView& w, const LinearRows& r) {
    const int k = linear_choice(w, r.rows);
    return k == 0 || k == 4 ? few_groups(w, r) : k == 1 ? many_groups(w, r, 2, 4) : k == 2 ? many_groups(w, r, 4, 4) : many_groups(w, r, 4, 8);
}

template <int W>
static void launch_few(const LinearArgs& a, const LinearRows& r, hipStream_t stream) {
    const dim3 grid((unsigned)few_groups(a.w, r));
#define CALL(END) launch(linear_few_kernel<END, W>, grid, dim3(64 * W), 0, stream, a)
    OHIP_LINEAR_END(CALL)
#undef CALL
}

constexpr int ROWS_W = 8;  // waves of linear_rows_kernel
constexpr int ROWS_STATICS = 16 * ROWS_W * (int)sizeof(float);  // its rows' sizes, which lie in the same memory
static int rows_lds(const LinearView& w, int rows) {
    const int codes = (rows < 16 ? rows : 16) * (int)linear_row_bytes(w.steps), sums = ROWS_W * (w.gated ? 2 : 1) * 1024;
    return codes > sums ? codes : sums;
}
static void launch_rows(const LinearArgs& a, const LinearRows& r, hipStream_t stream) {
    const dim3 grid((unsigned)few_groups(a.w, r));
#define CALL(END) launch(linear_rows_kernel<END, ROWS_W>, grid, dim3(64 * ROWS_W), rows_lds(a.w, r.rows), stream, a, r.x, r.x_stride)
    OHIP_LINEAR_END(CALL)
#undef CALL
}

template <int NT, int RT>
static void launch_many(const LinearArgs& a, const LinearRows& r, hipStream_t stream) {
    const dim3 grid((unsigned)many_groups(a.w, r, NT, RT));
#define CALL(END) launch(linear_many_kernel<NT, RT, END>, grid, dim3(256), 0, stream, a)
    OHIP_LINEAR_END(CALL)
#undef CALL
}

// The launch that is the fastest by a model of microseconds without the codes, fitted to measured products of 16 to 128 steps of inputs, 512 to
// 8192 outputs, 1 to 16384 rows and 1 to 64 experts. Over 92 such products, whose times profiles/ holds, the choice is 1.1 % over the
// fastest of the five launches on the mean and 25 % at most, where 16 rows go to 64 experts. The one for few rows reads weights and rows from
// the caches at 8 TB/s, 16 x 16 results at a time, but waits 1.2 for every 32 steps. The others take `each` for a stage of a workgroup by itself
// and `busy` where every compute unit has one, n times that for n: 64 x 128 results a wave are the least traffic, 32 x 64 start the soonest.
// 4096 x 4096 weights with codes: 128 rows 20.6 us (few: 25.9), 512 rows 25.4 (64 x 64: 29.7), 4096 rows 86 (32 x 64: 124), 16384 rows 350
// (64 x 64: 430).
int linear_choice(const LinearView& w, int rows) {
    const bool fits = rows_lds(w, rows) + ROWS_STATICS <= 65536;  // (what a launch has without an attribute)
    if (w.force >= 0) return w.force == 4 && !fits ? 0 : w.force;
    // Codes within the launch: where a workgroup has few of them to find and the workgroups run beside each other. A row of 2048 x 2048 6.2 ->
    // 5.1 us, two of 4000 x 4096 8.6 -> 7.8, three 8.6 -> 11.5; a row of 1024 x 16000 6.3 -> 8.4 (one launch behind another without a pause;
    // called from Python another 2 us less).
    const int n_tiles = w.tiles / (w.gated ? 2 : 1), most_tiles = rows < 16 * w.experts ? (rows < w.experts ? rows : w.experts) : (rows + 15) / 16;
    if (fits && (rows <= 2 || (size_t)rows * w.in <= 4096) && (size_t)n_tiles * most_tiles <= 512) return 4;
    const auto row_tiles = [&](int unit) {
        return w.experts == 1 ? (rows + unit - 1) / unit : rows / unit + (rows < w.experts ? rows : w.experts) * 0.5;
    };
    const double stages = (w.steps + 1) / 2, weights = (double)w.tiles * w.steps * 1024;
    const auto many = [&](int nt, int rt, double start, double each, double busy) {
        const double load = (w.tiles + 4 * nt - 1) / (4 * nt) * row_tiles(16 * rt) / 256 * busy;
        return start + stages * (load > each ? load : each);
    };
    const double waits = ((w.steps + 31) / 32) * 1.2, reads = row_tiles(16) * 2 * weights / 8e6;
    const double t[4] = {2.7 + (waits > reads ? waits : reads), many(2, 4, 4.4, 0.62, 0.61), many(4, 4, 3.2, 1.1, 0.89), many(4, 8, 10, 1.55, 1.3)};
    int best = 0;
    for (int i = 1; i < 4; ++i)
        if (t[i] < t[best]) best = i;
    return best;
}

hipError_t run_linear(const LinearView& w, const LinearRows& r, void* workspace, hipStream_t stream) {
    const LinearCodes c = linear_codes(w, r.x_rows, workspace);
    const int choice = linear_choice(w, r.rows);
    if (choice != 4) launch(linear_codes_kernel, dim3((unsigned)r.x_rows), dim3(256), 0, stream, r.x, r.x_stride, w.in, (int)linear_row_bytes(w.steps), c.scale, c.codes);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    LinearArgs a{w, c.scale, c.codes, r.index, r.starts, r.x_rows, r.rows, r.y, (size_t)r.rows * w.out * 4 > ((size_t)32 << 20)};
    if (w.act == 1) a.w.act_p0 = __builtin_inff();
    if (w.act == 3) a.w.act_p0 = 6.f;
    switch (choice) {
    case 0: {
        // eight waves share the inputs where the workgroups alone would leave compute units without work
        const double groups = (double)(w.tiles / (w.gated ? 2 : 1)) * ((r.rows + 15) / 16);
        if (groups < 1024 && w.steps >= 16) launch_few<8>(a, r, stream);
        else launch_few<4>(a, r, stream);
        break;
    }
    case 1: launch_many<2, 4>(a, r, stream); break;
    case 2: launch_many<4, 4>(a, r, stream); break;
    case 3: launch_many<4, 8>(a, r, stream); break;
    default: launch_rows(a, r, stream); break;
    }
    return hipGetLastError();
}

}  // namespace ohip
