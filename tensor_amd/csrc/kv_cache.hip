// The paged int8 cache of keys and values: tokens into it and out of it again (the layout is in kv_common.hpp).
//
// A workgroup owns the keys or the values of one head in one page. That is the unit that shares a scale, so the scale is found and
// used without leaving the workgroup, and a value tile's 16-byte pieces, which interleave tokens, have one writer.
#include "kv_common.hpp"

namespace ohip {

typedef float v4f __attribute__((ext_vector_type(4)));

// c * was / s rounded half away from zero, exactly: the product of a code and a float is exact in 64 bits, and so is the comparison with the
// middle between two codes, one fused multiply-add. inv = 1 / s, rounded: what it gives is off by one at most.
__device__ __forceinline__ int code_again(int c, double was, double s, double inv) {
    const double a = __builtin_fabs((double)c * was);
    double q = __builtin_floor(__builtin_fma(a, inv, 0.5));
    if (__builtin_fma(q - 0.5, -s, a) < 0.0) q -= 1.0;
    else if (__builtin_fma(q + 0.5, -s, a) >= 0.0) q += 1.0;
    const int i = min((int)q, 127);
    return c < 0 ? -i : i;
}

__device__ __forceinline__ int byte_of(unsigned v, int i) { return (int)(int8_t)(v >> (8 * i)); }

struct KvTile {
    KvSeq seq;
    int page;      // -1: not a page of the pool
    int position;  // of the block's first token (below 0: rows in front of the sequence)
    bool any;
};
// tile -> (sequence, block)
__device__ __forceinline__ KvTile kv_block_of(const KvBatch& b, int n_pages, int tile) {
    KvTile t;
    t.seq = kv_locate<KV_BLOCK, true, true>(b.starts, b.lengths, b.n_seqs, b.n_tokens, 1, tile);
    const int block = (t.seq.first >> 6) + t.seq.tile;
    t.any = t.seq.tile >= 0 && t.seq.count > 0 && block <= ((t.seq.length - 1) >> 6);
    t.position = block * KV_BLOCK;
    t.page = -1;
    if (t.any && block >= 0 && block < b.max_pages) {
        const int page = b.pages[(size_t)t.seq.index * b.max_pages + block];
        if ((unsigned)page < (unsigned)n_pages) t.page = page;
    }
    return t;
}

// A thread's unit is a square of 4 tokens x 4 dims: four float4 of rows on the float side, where neighbouring lanes read a row on, and
// four words on the cache's, each 4 dims of a token (keys) or 4 tokens of a dim (values). (A piece of 16 bytes a thread instead, 16
// floats of one token or dim, took 58 us for the append of 23 MB of codes and 92 us to read 27 MB back, single floats at a time.)
template <int KC, bool VALUES>
struct KvSquare {
    int token, dim;  // the first
    __device__ KvSquare(int unit) {
        // (values: four lanes have the tokens whose words are a piece of 16 bytes)
        if (VALUES) token = (unit & 3) * 16 + unit / (64 * KC) * 4, dim = (unit >> 2) % (16 * KC) * 4;
        else token = unit / (16 * KC) * 4, dim = unit % (16 * KC) * 4;
    }
    __device__ int at(int w) const { return VALUES ? kv_value_byte(token, dim + w) : kv_key_byte(token + w, dim); }  // word w's bytes
    __device__ static int row(int w, int e) { return VALUES ? e : w; }  // of the square, of word w's byte e
    __device__ static int column(int w, int e) { return VALUES ? w : e; }
};

// [rows][dims] of a square; rows outside [from, to) and dims behind the last are 0. `quads`: rows at multiples of 16 bytes, whole quads.
__device__ __forceinline__ void load_square(float (&v)[16], const float* __restrict__ rows, size_t stride, int token, int dim, int from, int to, int dims,
                                            bool quads) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const bool there = token + r >= from && token + r < to && dim < dims;
        const float* const p = rows + (ptrdiff_t)(token + r) * (ptrdiff_t)stride + dim;
        float4 f = {0.f, 0.f, 0.f, 0.f};
        if (quads) {
            if (there) f = *reinterpret_cast<const float4*>(p);
        } else if (there) {
            f.x = p[0];
            if (dim + 1 < dims) f.y = p[1];
            if (dim + 2 < dims) f.z = p[2];
            if (dim + 3 < dims) f.w = p[3];
        }
        v[4 * r] = f.x, v[4 * r + 1] = f.y, v[4 * r + 2] = f.z, v[4 * r + 3] = f.w;
    }
}

template <int KC, bool VALUES>
__device__ __forceinline__ void kv_append_block(const KvView& c, const KvTile& t, int head, const float* __restrict__ x, size_t stride) {
    typedef KvSquare<KC, VALUES> Square;
    __shared__ float most_of[4];
    const int tid = (int)threadIdx.x;
    const int from = max(t.seq.first - t.position, 0);        // the block's first new token (0: none is older)
    const int to = min(t.seq.length - t.position, KV_BLOCK);  // behind its last
    // row of slot i: begin + (position + i - first)
    const float* const rows = x + ((ptrdiff_t)t.seq.begin + t.position - t.seq.first) * (ptrdiff_t)stride + (size_t)head * c.dim;
    const bool quads = c.dim % 4 == 0 && stride % 4 == 0 && ((size_t)x & 15) == 0;
    float v[KC][16];
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
        const Square p(tid + 256 * u);
        load_square(v[u], rows, stride, p.token, p.dim, from, to, c.dim, quads);
    }
    // (the page's number is on its way with the rows: a call for one token of each sequence is made of such waits)
    if (t.page < 0) return;
    int8_t* const codes = (VALUES ? c.v : c.k) + c.at(t.page, head);
    float* const scale = (VALUES ? c.vs : c.ks) + (size_t)t.page * c.heads + head;
    float was = from > 0 ? *scale : 0.f;
#pragma unroll
    for (int u = 0; u < KC; ++u) most = fmaxf(most, largest_size(v[u]));
#pragma unroll
    for (int m = 32; m; m >>= 1) most = fmaxf(most, __shfl_xor(most, m));
    if ((tid & 63) == 0) most_of[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3]));
    if (!(was >= KV_LEAST_SCALE && was < __builtin_inff())) was = 0.f;
    const float s = fmaxf(was, scale_of(most));
    const bool again = s > was;  // the older tokens' codes change
    const Coder coder(s);
    // The older tokens' codes in the new scale, word by word: in a loop, as it is seldom run and would be most of the launch's code.
    // (A thread's words are those of its squares: what it leaves here it finds below.)
    if (again && from > 0) {
        const double inv64 = 1.0 / (double)s;
#pragma unroll 1
        for (int n = 0; n < 4 * KC; ++n) {
            const Square p(tid + 256 * (n >> 2));
            if (p.token + Square::row(n & 3, 0) >= from) continue;
            unsigned* const at = reinterpret_cast<unsigned*>(codes + p.at(n & 3));
            unsigned word = *at;
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {  // (the byte in front leaves, its code comes in behind)
                const int c = byte_of(word, 0);
                const int code = p.token + Square::row(n & 3, e) >= from ? c : was > 0.f ? code_again(c, was, s, inv64) : 0;
                word = (word >> 8) | ((unsigned)(code & 0xff) << 24);
            }
            *at = word;
        }
    }
    // (tokens in front of a word's first new one keep their bytes)
    const auto older = [&](const Square& p, int w) {
        unsigned mask = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) mask |= p.token + Square::row(w, e) < from ? 0xffu << (8 * e) : 0u;
        return mask;
    };
    bool doubtful = false;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
        const Square p(tid + 256 * u);
        if (p.token >= to || p.token + 4 <= from) continue;  // no new token
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = v[u][4 * Square::row(w, e) + Square::column(w, e)];
            unsigned now = (unsigned)coder.word(f[0], f[1], f[2], f[3], doubtful);
            unsigned* const at = reinterpret_cast<unsigned*>(codes + p.at(w));
            if (p.token < from) {
                const unsigned mask = older(p, w);
                now = (*at & mask) | (now & ~mask);
            }
            *at = now;
        }
    }
    if (doubtful) {  // (its words once more, one after another)
#pragma unroll 1
        for (int n = 0; n < 4 * KC; ++n) {
            const Square p(tid + 256 * (n >> 2));
            if (p.token >= to || p.token + 4 <= from) continue;
            unsigned* const at = reinterpret_cast<unsigned*>(codes + p.at(n & 3));
            unsigned now = 0;
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
                const int slot = p.token + Square::row(n & 3, e), d = p.dim + Square::column(n & 3, e);
                const float f = slot >= from && slot < to && d < c.dim ? rows[(ptrdiff_t)slot * (ptrdiff_t)stride + d] : 0.f;
                now |= (unsigned)coder.exact(f) << (8 * e);
            }
            const unsigned mask = older(p, n & 3);
            *at = (*at & mask) | (now & ~mask);
        }
    }
    if (tid == 0) *scale = s;
}

template <int KC>
__global__ void __launch_bounds__(256) kv_append_kernel(KvView c, KvBatch b, const float* __restrict__ k, size_t k_stride,
                                                        const float* __restrict__ v, size_t v_stride) {
    const int parts = 2 * c.heads, part = (int)(blockIdx.x % (unsigned)parts);
    const KvTile t = kv_block_of(b, c.n_pages, (int)(blockIdx.x / (unsigned)parts));
    if (!t.any) return;
    if (part < c.heads) kv_append_block<KC, false>(c, t, part, k, k_stride);
    else kv_append_block<KC, true>(c, t, part - c.heads, v, v_stride);
}

template <int KC, bool VALUES>
__device__ __forceinline__ void kv_read_block(const KvView& c, const KvTile& t, int head, float* __restrict__ x) {
    typedef KvSquare<KC, VALUES> Square;
    const int tid = (int)threadIdx.x;
    const size_t stride = (size_t)c.heads * c.dim;
    const int8_t* const codes = (VALUES ? c.v : c.k) + (t.page < 0 ? 0 : c.at(t.page, head));
    const float s = t.page < 0 ? 0.f : (VALUES ? c.vs : c.ks)[(size_t)t.page * c.heads + head];
    const int from = max(t.seq.first - t.position, 0), to = min(t.seq.length - t.position, KV_BLOCK);
    float* const rows = x + ((ptrdiff_t)t.seq.begin + t.position - t.seq.first) * (ptrdiff_t)stride + (size_t)head * c.dim;
    const bool quads = c.dim % 4 == 0 && ((size_t)x & 15) == 0;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
        const Square p(tid + 256 * u);
        if (p.token >= to || p.token + 4 <= from || p.dim >= c.dim) continue;
        float v[4][4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            unsigned word = 0;
            if (t.page >= 0) word = *reinterpret_cast<const unsigned*>(codes + p.at(w));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[Square::row(w, e)][Square::column(w, e)] = t.page < 0 ? 0.f : __fmul_rn((float)byte_of(word, e), s);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (p.token + r < from || p.token + r >= to) continue;
            float* const to_row = rows + (ptrdiff_t)(p.token + r) * (ptrdiff_t)stride + p.dim;
            if (quads) {  // (four times the codes, and seldom read again by the GPU: not kept in the caches. 27 MB of codes 38.5 -> 21.8 us)
                const v4f f = {v[r][0], v[r][1], v[r][2], v[r][3]};
                __builtin_nontemporal_store(f, reinterpret_cast<v4f*>(to_row));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (p.dim + e < c.dim) to_row[e] = v[r][e];
            }
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
