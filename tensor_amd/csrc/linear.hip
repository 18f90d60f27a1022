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
    int8_t* codes;  // [x_rows][steps * 64]
};
static LinearCodes linear_codes(const LinearView& w, int x_rows, void* workspace) {
    LinearCodes c;
    c.scale = (float*)workspace;
    c.codes = (int8_t*)workspace + ((size_t)x_rows * 4 + 255) / 256 * 256;
    return c;
}
size_t linear_workspace_bytes(const LinearView& w, int x_rows) { return ((size_t)x_rows * 4 + 255) / 256 * 256 + (size_t)x_rows * w.steps * 64; }

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
__device__ __forceinline__ int codes_of_quad(const float4& f, float s, float inv) {
    if (!(s > 0.f)) return 0;
    return (code_of(f.x, s, inv) & 0xff) | ((code_of(f.y, s, inv) & 0xff) << 8) | ((code_of(f.z, s, inv) & 0xff) << 16) | (code_of(f.w, s, inv) << 24);
}
__device__ __forceinline__ float most_of_quad(const float4& f) {
    return fmaxf(fmaxf(finite_size(f.x), finite_size(f.y)), fmaxf(finite_size(f.z), finite_size(f.w)));
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
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < KEPT; ++u) most = fmaxf(most, most_of_quad(kept[u]));
    for (int d = 4 * tid + 1024 * KEPT; d < in; d += 1024) most = fmaxf(most, most_of_quad(row_quad(row, d, in, quads)));
#pragma unroll
    for (int m = 32; m; m >>= 1) most = fmaxf(most, __shfl_xor(most, m));
    if ((tid & 63) == 0) most_of[tid >> 6] = most;
    __syncthreads();
    const float s = scale_of(fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3])));
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    if (tid == 0) scale[blockIdx.x] = s;
    int* const to = reinterpret_cast<int*>(codes + (size_t)blockIdx.x * padded);
#pragma unroll
    for (int u = 0; u < KEPT; ++u)
        if (4 * tid + 1024 * u < padded) to[tid + 256 * u] = codes_of_quad(kept[u], s, inv);
    for (int d = 4 * tid + 1024 * KEPT; d < padded; d += 1024) to[d >> 2] = codes_of_quad(row_quad(row, d, in, quads), s, inv);
}

struct LinearArgs {
    LinearView w;
    const float* scale;
    const int8_t* codes;
    const int32_t *index, *starts;
    int x_rows, rows;
    float* y;
};

// Expert and rows of a tile of `unit` rows: [begin, end), empty where the tile is behind its expert's rows.
struct LinearTile {
    int expert, begin, end;
};
__device__ __forceinline__ LinearTile linear_tile(const LinearArgs& a, int tile, int unit) {
    LinearTile t;
    if (!a.starts) {
        t.expert = 0, t.begin = tile * unit, t.end = min(t.begin + unit, a.rows);
        return t;
    }
    t.expert = kv_find(a.starts, a.w.experts, a.rows, 1, unit, 1, tile);
    const int from = min(max(a.starts[t.expert], 0), a.rows), to = min(max(a.starts[t.expert + 1], from), a.rows);
    const int n = tile - kv_tile_base(a.starts, t.expert, a.rows, 1, unit, 1);
    t.begin = n < 0 ? to : min(from + n * unit, to);
    t.end = min(t.begin + unit, to);
    return t;
}
static int linear_row_tiles(const LinearView& w, const LinearRows& r, int unit) {
    return r.starts ? r.rows / unit + w.experts : (r.rows + unit - 1) / unit;
}

// Row of x behind a sorted row (an index outside of x: -1).
__device__ __forceinline__ int linear_source(const LinearArgs& a, int row) {
    const int i = a.index ? a.index[row] : row;
    return (unsigned)i < (unsigned)a.x_rows ? i : -1;
}

// Four consecutive outputs of one row.
template <bool GATED>
__device__ __forceinline__ void linear_store(const LinearArgs& a, int expert, int n_tile, int row, float xs, const v4i& acc, const v4i& acc_up) {
    const int g = (int)(threadIdx.x >> 4) & 3;
    const size_t at = ((size_t)expert * a.w.tiles + (size_t)n_tile * (GATED ? 2 : 1)) * 16 + g * 4;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float b = a.w.bias ? a.w.bias[at + e] : 0.f;
        v[e] = __fmaf_rn((float)acc[e], __fmul_rn(xs, a.w.scale[at + e]), b);
        if constexpr (GATED) {
            const float bu = a.w.bias ? a.w.bias[at + 16 + e] : 0.f;
            const float up = __fmaf_rn((float)acc_up[e], __fmul_rn(xs, a.w.scale[at + 16 + e]), bu);
            v[e] = __fmul_rn(__fdiv_rn(v[e], __fadd_rn(1.f, __expf(-v[e]))), up);
        } else v[e] = activate(v[e], a.w.act, a.w.act_p0);
    }
    const int n = n_tile * 16 + g * 4;
    float* const to = a.y + (size_t)row * a.w.out + n;
    if (a.w.out % 4 == 0 && ((size_t)a.y & 15) == 0) {
        if (n < a.w.out) *reinterpret_cast<float4*>(to) = {v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < a.w.out) to[e] = v[e];
    }
}

// 16 outputs (gated: 16 of either half) x 16 RT rows a workgroup, the inputs dealt to its four waves, whose sums meet in LDS. Both
// operands come straight from memory in lane order; this is the launch for few rows, where reading the weights is the work.
template <int RT, bool GATED>
__global__ void __launch_bounds__(256) linear_few_kernel(LinearArgs a) {
    constexpr int G = GATED ? 2 : 1;
    __shared__ v4i sums[4][G * RT][64];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const unsigned n_tiles = (unsigned)a.w.tiles / G;
    const int n_tile = (int)(blockIdx.x % n_tiles);
    const LinearTile t = linear_tile(a, (int)(blockIdx.x / n_tiles), 16 * RT);
    if (t.begin >= t.end) return;
    const size_t step_bytes = (size_t)a.w.steps * 64;
    const int8_t* const w = a.w.w + ((size_t)t.expert * a.w.tiles + (size_t)n_tile * G) * a.w.steps * 1024 + lane * 16;
    const int8_t* x[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int src = linear_source(a, min(t.begin + i * 16 + (lane & 15), t.end - 1));
        x[i] = a.codes + (size_t)max(src, 0) * step_bytes + (lane >> 4) * 16;
    }
    v4i acc[G][RT] = {};
    for (int s = wave; s < a.w.steps; s += 4) {
        v4i b[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) b[i] = *reinterpret_cast<const v4i*>(x[i] + s * 64);
#pragma unroll
        for (int h = 0; h < G; ++h) {
            const v4i k = *reinterpret_cast<const v4i*>(w + ((size_t)h * a.w.steps + s) * 1024);
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[h][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, b[i], acc[h][i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
        for (int i = 0; i < RT; ++i) sums[wave][h * RT + i][lane] = acc[h][i];
    __syncthreads();
    if (wave >= RT) return;
    v4i sum[2] = {};
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
        for (int n = 0; n < 4; ++n) sum[h] += sums[n][h * RT + wave][lane];
    const int row = t.begin + wave * 16 + (lane & 15);
    if (row >= t.end) return;
    const int src = linear_source(a, row);
    linear_store<GATED>(a, t.expert, n_tile, row, src < 0 ? 0.f : a.scale[src], sum[0], sum[1]);
}

template <int RT>
static void launch_few(const LinearArgs& a, const LinearRows& r, hipStream_t stream) {
    const dim3 grid((unsigned)(a.w.tiles / (a.w.gated ? 2 : 1)) * (unsigned)linear_row_tiles(a.w, r, 16 * RT));
    if (a.w.gated) launch(linear_few_kernel<RT, true>, grid, dim3(256), 0, stream, a);
    else launch(linear_few_kernel<RT, false>, grid, dim3(256), 0, stream, a);
}

hipError_t run_linear(const LinearView& w, const LinearRows& r, void* workspace, hipStream_t stream) {
    const LinearCodes c = linear_codes(w, r.x_rows, workspace);
    if (r.x_rows) launch(linear_codes_kernel, dim3((unsigned)r.x_rows), dim3(256), 0, stream, r.x, r.x_stride, w.in, w.steps * 64, c.scale, c.codes);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const LinearArgs a{w, c.scale, c.codes, r.index, r.starts, r.x_rows, r.rows, r.y};
    // rows of a tile: few where an expert has few (the tiles of an expert without rows end at once)
    if (r.rows <= 16 * w.experts) launch_few<1>(a, r, stream);
    else if (r.rows <= 32 * w.experts) launch_few<2>(a, r, stream);
    else launch_few<4>(a, r, stream);
    return hipGetLastError();
}

}  // namespace ohip
