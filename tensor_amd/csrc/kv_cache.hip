// The paged int8 cache of keys and values: tokens into it and out of it again (the layout is in kv_common.hpp).
//
// A workgroup owns the keys or the values of one head in one page. That is the unit that shares a scale, so the scale is found and
// used without leaving the workgroup, and a value tile's 16-byte pieces, which interleave tokens, have one writer.
#include "kv_common.hpp"

namespace ohip {

// c * was / s rounded half away from zero, exactly: the product of a code and a float is exact in 64 bits, the comparison with the
// middle between two codes one fused multiply-add.
__device__ __forceinline__ int code_again(int c, float was, float s) {
    const double a = __builtin_fabs((double)c * (double)was), d = (double)s;
    double q = __builtin_floor(a / d + 0.5);
    if (__builtin_fma(q - 0.5, -d, a) < 0.0) q -= 1.0;
    else if (__builtin_fma(q + 0.5, -d, a) >= 0.0) q += 1.0;
    const int i = min((int)q, 127);
    return c < 0 ? -i : i;
}

__device__ __forceinline__ int byte_of(ohip_v4i v, int i) { return (int)(int8_t)(v[i >> 2] >> (8 * (i & 3))); }
__device__ __forceinline__ void set_byte(ohip_v4i& v, int i, int c) {
    const int at = 8 * (i & 3);
    v[i >> 2] = (int)(((unsigned)v[i >> 2] & ~(0xffu << at)) | ((unsigned)(c & 0xff) << at));
}

struct KvTile {
    KvSeq seq;
    int page;      // -1: not a page of the pool
    int position;  // of the block's first token (below 0: rows in front of the sequence)
    bool any;
};
// tile -> (sequence, block)
__device__ __forceinline__ KvTile kv_block_of(const KvBatch& b, int n_pages, int tile) {
    const int i = kv_find(b.starts, b.n_seqs, b.n_tokens, 1, KV_BLOCK, 2, tile);
    KvTile t;
    t.seq = kv_sequence(b, i);
    const int block = (t.seq.first >> 6) + (tile - kv_tile_base(b.starts, i, b.n_tokens, 1, KV_BLOCK, 2));
    t.any = tile >= kv_tile_base(b.starts, i, b.n_tokens, 1, KV_BLOCK, 2) && t.seq.count > 0 && block <= ((t.seq.length - 1) >> 6);
    t.position = block * KV_BLOCK;
    t.page = -1;
    if (t.any && block >= 0 && block < b.max_pages) {
        const int page = b.pages[(size_t)i * b.max_pages + block];
        if ((unsigned)page < (unsigned)n_pages) t.page = page;
    }
    return t;
}

// 16 tokens or dims of a thread: keys are dealt as (token, 16 dims), read 64 bytes at a time, values as (16 tokens, dim), each
// token's row read by neighbouring lanes.
template <int KC, bool VALUES>
struct KvPiece {
    int token, dim;  // the first
    __device__ KvPiece(int unit) {
        if (VALUES) dim = unit % (64 * KC), token = (unit / (64 * KC)) * 4;
        else dim = (unit % (4 * KC)) * 16, token = unit / (4 * KC);
    }
    __device__ int slot(int e) const { return VALUES ? token + 16 * (e >> 2) + (e & 3) : token; }
    __device__ int column(int e) const { return VALUES ? dim : dim + e; }
    __device__ int byte() const { return VALUES ? kv_value_byte(token, dim) : kv_key_byte(token, dim); }
};

template <int KC, bool VALUES>
__device__ __forceinline__ void kv_append_block(const KvView& c, const KvTile& t, int head, const float* __restrict__ x, size_t stride) {
    __shared__ float most_of[4];
    const int tid = (int)threadIdx.x;
    int8_t* const codes = (VALUES ? c.v : c.k) + c.at(t.page, head);
    float* const scale = (VALUES ? c.vs : c.ks) + (size_t)t.page * c.heads + head;
    const int from = max(t.seq.first - t.position, 0);                    // the block's first new token (0: none is older)
    const int to = min(t.seq.length - t.position, KV_BLOCK);              // behind its last
    // row of slot i: begin + (position + i - first)
    const float* const rows = x + ((ptrdiff_t)t.seq.begin + t.position - t.seq.first) * (ptrdiff_t)stride + (size_t)head * c.dim;
    float v[KC][16];
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
        const KvPiece<KC, VALUES> p(tid + 256 * u);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int s = p.slot(e), d = p.column(e);
            v[u][e] = s >= from && s < to && d < c.dim ? rows[(ptrdiff_t)s * (ptrdiff_t)stride + d] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) most = fmaxf(most, finite_size(v[u][e]));
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) most = fmaxf(most, __shfl_xor(most, m));
    if ((tid & 63) == 0) most_of[tid >> 6] = most;
    float was = from > 0 ? *scale : 0.f;
    __syncthreads();
    most = fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3]));
    if (!(was >= KV_LEAST_SCALE && was < __builtin_inff())) was = 0.f;
    const float s = fmaxf(was, scale_of(most));
    const bool again = s > was;  // the older tokens' codes change
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
        const KvPiece<KC, VALUES> p(tid + 256 * u);
        const int lo = p.slot(0);  // its first token
        bool fresh = false;
#pragma unroll
        for (int e = 0; e < 16; e += 4) fresh |= p.slot(e + 3) >= from && p.slot(e) < to;
        if (lo >= to || !(fresh || (again && lo < from))) continue;
        ohip_v4i* const at = reinterpret_cast<ohip_v4i*>(codes + p.byte());
        ohip_v4i w = {0, 0, 0, 0};
        if (from > 0 && lo < from) w = *at;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int slot = p.slot(e);
            int code = 0;
            if (slot < from) code = !again ? byte_of(w, e) : was > 0.f ? code_again(byte_of(w, e), was, s) : 0;
            else if (slot < to && s > 0.f) code = code_of(v[u][e], s, inv);
            set_byte(w, e, code);
        }
        *at = w;
    }
    if (tid == 0) *scale = s;
}

template <int KC>
__global__ void __launch_bounds__(256) kv_append_kernel(KvView c, KvBatch b, const float* __restrict__ k, size_t k_stride,
                                                        const float* __restrict__ v, size_t v_stride) {
    const int parts = 2 * c.heads, part = (int)(blockIdx.x % (unsigned)parts);
    const KvTile t = kv_block_of(b, c.n_pages, (int)(blockIdx.x / (unsigned)parts));
    if (!t.any || t.page < 0) return;
    if (part < c.heads) kv_append_block<KC, false>(c, t, part, k, k_stride);
    else kv_append_block<KC, true>(c, t, part - c.heads, v, v_stride);
}

template <int KC, bool VALUES>
__device__ __forceinline__ void kv_read_block(const KvView& c, const KvTile& t, int head, float* __restrict__ x) {
    const int tid = (int)threadIdx.x;
    const size_t stride = (size_t)c.heads * c.dim;
    const int8_t* const codes = (VALUES ? c.v : c.k) + (t.page < 0 ? 0 : c.at(t.page, head));
    const float s = t.page < 0 ? 0.f : (VALUES ? c.vs : c.ks)[(size_t)t.page * c.heads + head];
    const int from = max(t.seq.first - t.position, 0), to = min(t.seq.length - t.position, KV_BLOCK);
    float* const rows = x + ((ptrdiff_t)t.seq.begin + t.position - t.seq.first) * (ptrdiff_t)stride + (size_t)head * c.dim;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
        const KvPiece<KC, VALUES> p(tid + 256 * u);
        ohip_v4i w = {0, 0, 0, 0};
        if (t.page >= 0) w = *reinterpret_cast<const ohip_v4i*>(codes + p.byte());
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int slot = p.slot(e), d = p.column(e);
            if (slot >= from && slot < to && d < c.dim) rows[(ptrdiff_t)slot * (ptrdiff_t)stride + d] = t.page < 0 ? 0.f : __fmul_rn((float)byte_of(w, e), s);
        }
    }
}

template <int KC>
__global__ void __launch_bounds__(256) kv_read_kernel(KvView c, KvBatch b, float* __restrict__ k, float* __restrict__ v) {
    const int parts = 2 * c.heads, part = (int)(blockIdx.x % (unsigned)parts);
    const KvTile t = kv_block_of(b, c.n_pages, (int)(blockIdx.x / (unsigned)parts));
    if (!t.any) return;
    if (part < c.heads) {
        if (k) kv_read_block<KC, false>(c, t, part, k);
    } else if (v) kv_read_block<KC, true>(c, t, part - c.heads, v);
}

// blocks that the rows of a batch can touch, at most
static unsigned kv_block_tiles(const KvBatch& b) { return (unsigned)b.n_tokens / KV_BLOCK + 2u * (unsigned)b.n_seqs; }

#define OHIP_KV_CHUNKS(CALL) \
    switch (c.chunks) {      \
    case 1: CALL(1); break;  \
    case 2: CALL(2); break;  \
    case 3: CALL(3); break;  \
    default: CALL(4); break; \
    }

hipError_t run_kv_append(const KvView& c, const KvBatch& b, const float* k, size_t k_stride, const float* v, size_t v_stride,
                         hipStream_t stream) {
    const dim3 grid(kv_block_tiles(b) * 2u * (unsigned)c.heads);
#define CALL(KC) launch(kv_append_kernel<KC>, grid, dim3(256), 0, stream, c, b, k, k_stride, v, v_stride)
    OHIP_KV_CHUNKS(CALL)
#undef CALL
    return hipGetLastError();
}

hipError_t run_kv_read(const KvView& c, const KvBatch& b, float* k, float* v, hipStream_t stream) {
    const dim3 grid(kv_block_tiles(b) * 2u * (unsigned)c.heads);
#define CALL(KC) launch(kv_read_kernel<KC>, grid, dim3(256), 0, stream, c, b, k, v)
    OHIP_KV_CHUNKS(CALL)
#undef CALL
    return hipGetLastError();
}

}  // namespace ohip
