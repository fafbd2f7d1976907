// Kernels that keep the 8-bit cache: words of the book, rows in (append), numbers out (read), pages copied and tokens moved together (keep).
#pragma once

#include "wd_kv_layout.cuh"

namespace wd {

// ---- words of the book, by value: ordered by the stream, and no staging buffer that a later call could overwrite -----------------
template <int N>
struct KvWords {
    int n, pad;
    int2 w[N];          // offset, value
};
template <int N>
__global__ void __launch_bounds__(256) kv_words_kernel(const __grid_constant__ KvWords<N> P, int *book) {
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) book[P.w[i].x] = P.w[i].y;
}
template <int N>
struct KvRun {
    int n, offset;
    int w[N];           // values of a run
};
template <int N>
__global__ void __launch_bounds__(256) kv_run_kernel(const __grid_constant__ KvRun<N> P, int *to) {
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) to[P.offset + i] = P.w[i];
}

// ---- append ---------------------------------------------------------------------------------------------------------------
// A block takes the step's tokens that lie in one page, one kv head, keys (blockIdx.z = 0) or values. Two passes over its rows: the largest
// magnitude, from which the scale follows, then the codes (the rows come from the caches the second time). A page that held tokens before keeps its
// scale unless the new ones need a larger one; then the codes that are there are rounded anew.
struct KvAppend {
    uint8_t *pool;              // of the layer
    float *scales;              // of the layer
    const int *book;
    const int *table;
    const void *rows[2];
    long long stride[2];
    unsigned *status;
    int type;
    KvShape s;
};
constexpr int kAppendThreads = 128;

template <bool E4M3>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ KvAppend P) {
    __shared__ float part[kAppendThreads / 32];
    __shared__ int bad_any;
    const int n_seq = P.book[0], n_items = P.book[2], tid = threadIdx.x, h = blockIdx.y, kv = blockIdx.z, D = P.s.head_dim;
    const int *entries = P.book + kKvHead;
    const int page_tokens = 1 << P.s.page_shift;
    const size_t stride = static_cast<size_t>(P.stride[kv]);
    const void *rows = P.rows[kv];
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const int *e = entries + kv_entry_of_item(entries, n_seq, item) * kKvStepWords;
        const int seq = e[0], row0 = e[1], count = e[2], length = e[3], begin = length - count;
        const int logical = (begin >> P.s.page_shift) + item - e[4], page0 = logical << P.s.page_shift;
        const int a = max(begin - page0, 0), b = min(length - page0, page_tokens);       // the step's tokens in this page: a .. b - 1
        const int page = P.table[static_cast<size_t>(seq) * P.s.max_pages + logical];
        const size_t first = static_cast<size_t>(row0 + page0 + a - begin);
        uint8_t *base = P.pool + static_cast<size_t>(page) * kv_page_bytes(P.s) + h * kv_head_bytes(P.s) + kv * kv_half_bytes(P.s);
        float *scale = P.scales + (static_cast<size_t>(page) * P.s.kv_heads + h) * 2 + kv;
        const float s0 = a > 0 ? *scale : 0.0f;
        const size_t col = static_cast<size_t>(h) * D;
        // the largest finite magnitude
        float top = 0.0f;
        int bad = 0;
        const int total = (b - a) * D;
#pragma unroll 4
        for (int i = tid; i < total; i += kAppendThreads) {
            const int t = i / D, d = i - t * D;
            const float x = fabsf(row_load(rows, P.type, (first + t) * stride + col + d));
            if (x <= 3.402823466e38f) top = fmaxf(top, x);
            else bad = 1;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (tid == 0) bad_any = 0;
        __syncthreads();
        if ((tid & 31) == 0) part[tid >> 5] = top;
        if (bad) bad_any = 1;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; ++w) top = fmaxf(top, part[w]);
        if (tid == 0 && bad_any) atomicOr(P.status, kKvNonFinite);
        const float need = top > 0.0f ? fmaxf(__fdiv_rn(top, E4M3 ? 448.0f : 127.0f), kKvLeastScale) : 0.0f;
        const float s1 = fmaxf(s0, need), r = s1 > 0.0f ? __fdiv_rn(1.0f, s1) : 0.0f;
        if (a > 0 && s1 != s0) {        // the codes of the tokens 0 .. a - 1 under the larger scale
            const int vecs = ((a + kKvSub - 1) / kKvSub) * D;
            for (int i = tid; i < vecs; i += kAppendThreads) {
                const int sub = i / D, v = i - sub * D;
                uint4 *p = reinterpret_cast<uint4 *>(base + sub * kv_sub_bytes(D)) + v;
                uint4 x = *p;
                uint8_t *c = reinterpret_cast<uint8_t *>(&x);
                const int cw = kv_cw(D), token = (v * 16 % (16 * cw)) / cw;      // (keys)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (sub * kKvSub + (kv ? kv_v_token(v, j) : token) < a) c[j] = static_cast<uint8_t>(kv_recode<E4M3>(c[j], s0, s1));
                *p = x;
            }
        }
        __syncthreads();        // the values' old and new tokens may share 16 bytes
        if (kv == 0) {
            const int per = D / 16, vecs = (b - a) * per;
            for (int i = tid; i < vecs; i += kAppendThreads) {
                const int t = i / per, k = (i - t * per) * 16, token = a + t;
                const size_t src = (first + t) * stride + col + k;
                uint4 x;
                uint8_t *c = reinterpret_cast<uint8_t *>(&x);
#pragma unroll
                for (int j = 0; j < 16; ++j) c[j] = static_cast<uint8_t>(kv_code<E4M3>(row_load(rows, P.type, src + j), s1, r));
                *reinterpret_cast<uint4 *>(base + (token / kKvSub) * kv_sub_bytes(D) + kv_k_offset(D, token % kKvSub, k)) = x;
            }
        } else {
            const int sub0 = a / kKvSub, subs = (b - 1) / kKvSub + 1 - sub0;
            for (int i = tid; i < subs * D; i += kAppendThreads) {
                const int sub = sub0 + i / D, v = i % D, lo = a - sub * kKvSub, hi = b - sub * kKvSub;
                uint8_t *to = base + sub * kv_sub_bytes(D) + v * 16;
                uint4 x;
                uint8_t *c = reinterpret_cast<uint8_t *>(&x);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int token = kv_v_token(v, j);
                    if (token >= lo && token < hi)
                        c[j] = static_cast<uint8_t>(kv_code<E4M3>(row_load(rows, P.type, (first + token - lo) * stride + col + kv_v_element(v, j)), s1, r));
                }
                if (lo <= 0 && hi >= kKvSub) {
                    *reinterpret_cast<uint4 *>(to) = x;
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (kv_v_token(v, j) >= lo && kv_v_token(v, j) < hi) to[j] = c[j];
                }
            }
        }
        if (tid == 0) *scale = s1;
        __syncthreads();
    }
}

// ---- read -----------------------------------------------------------------------------------------------------------------
// Tokens first .. first + count - 1 of sequences as numbers, rows one after the other: [layer][row][kv head][D]. A block takes a sub-block of
// 16 tokens, one head, keys or values of one layer.
struct KvReadEntry {
    int seq, first, count, row0, item0;         // items: sub-blocks that the range touches
};
constexpr int kReadEntries = 100;
struct KvRead {
    const uint8_t *pool;        // of the first layer
    const float *scales;
    const int *table;
    void *out[2];
    size_t pool_layer, scales_layer, out_layer;         // bytes, floats, elements from a layer to the next
    int type, n, n_rows_pad;
    KvShape s;
    KvReadEntry e[kReadEntries];
};
constexpr int kReadThreads = 128;

template <bool E4M3>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const __grid_constant__ KvRead P) {
    const int item = blockIdx.x, h = blockIdx.y % P.s.kv_heads, layer = blockIdx.y / P.s.kv_heads, kv = blockIdx.z, D = P.s.head_dim, tid = threadIdx.x;
    if (P.out[kv] == nullptr) return;
    int lo = 0, hi = P.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (P.e[mid].item0 <= item) lo = mid;
        else hi = mid - 1;
    }
    const KvReadEntry e = P.e[lo];
    const int sub = e.first / kKvSub + item - e.item0, t0 = sub * kKvSub;
    const int a = max(e.first - t0, 0), b = min(e.first + e.count - t0, kKvSub), shift = P.s.page_shift;
    const int page = P.table[static_cast<size_t>(e.seq) * P.s.max_pages + (t0 >> shift)];
    const uint8_t *base = P.pool + layer * P.pool_layer + static_cast<size_t>(page) * kv_page_bytes(P.s) + h * kv_head_bytes(P.s) +
                          ((t0 & ((1 << shift) - 1)) / kKvSub) * kv_sub_bytes(D) + kv * kv_half_bytes(P.s);
    const float s = P.scales[layer * P.scales_layer + (static_cast<size_t>(page) * P.s.kv_heads + h) * 2 + kv];
    const size_t pitch = static_cast<size_t>(P.s.kv_heads) * D;
    const size_t out0 = layer * P.out_layer + static_cast<size_t>(e.row0 + t0 - e.first) * pitch + static_cast<size_t>(h) * D;     // (of token 0, which may lie in front of the rows)
    if (kv == 0) {
        const int per = D / 16;
        for (int i = a * per + tid; i < b * per; i += kReadThreads) {
            const int t = i / per, k = (i - t * per) * 16;
            const uint4 x = *reinterpret_cast<const uint4 *>(base + kv_k_offset(D, t, k));
            const uint8_t *c = reinterpret_cast<const uint8_t *>(&x);
            const size_t to = out0 + t * pitch + k;
#pragma unroll
            for (int j = 0; j < 16; ++j) row_store(P.out[0], P.type, to + j, __fmul_rn(kv_value<E4M3>(c[j]), s));
        }
    } else {
        for (int v = tid; v < D; v += kReadThreads) {
            const uint4 x = *reinterpret_cast<const uint4 *>(base + v * 16);
            const uint8_t *c = reinterpret_cast<const uint8_t *>(&x);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int token = kv_v_token(v, j);
                if (token >= a && token < b) row_store(P.out[1], P.type, out0 + token * pitch + kv_v_element(v, j), __fmul_rn(kv_value<E4M3>(c[j]), s));
            }
        }
    }
}

// ---- copy of pages (a page that several sequences hold, before one of them writes into it) -----------------------------------------
constexpr int kCopyPairs = 200;
struct KvCopy {
    uint8_t *pool;
    float *scales;
    size_t pool_layer, scales_layer, page_bytes;
    int n, n_layers, page_scales;
    int2 pair[kCopyPairs];      // from, to
};
__global__ void __launch_bounds__(256) kv_copy_kernel(const __grid_constant__ KvCopy P) {
    const int2 pr = P.pair[blockIdx.y];
    const size_t vecs = P.page_bytes / 16;
    const int layer = blockIdx.z;
    const uint4 *from = reinterpret_cast<const uint4 *>(P.pool + layer * P.pool_layer + pr.x * P.page_bytes);
    uint4 *to = reinterpret_cast<uint4 *>(P.pool + layer * P.pool_layer + pr.y * P.page_bytes);
#pragma unroll 4
    for (size_t i = blockIdx.x * 256 + threadIdx.x; i < vecs; i += static_cast<size_t>(gridDim.x) * 256) to[i] = from[i];
    if (blockIdx.x == 0) {
        float *sc = P.scales + layer * P.scales_layer;
        for (int i = threadIdx.x; i < P.page_scales; i += 256) sc[static_cast<size_t>(pr.y) * P.page_scales + i] = sc[static_cast<size_t>(pr.x) * P.page_scales + i];
    }
}

// ---- keep -----------------------------------------------------------------------------------------------------------------
// Of a sequence's tokens from `first` on those of `index` stay and move together. A block builds one page, one head, keys or values of one layer:
// its tokens come from pages behind it (or itself), its scale is the largest of theirs, codes of smaller ones are rounded anew. Pages that are built
// into new pages are independent of one another (gridDim.x = pages); where there are none to be had, a block walks over the pages in their order,
// reading all of a page's tokens before it writes (gridDim.x = 1).
struct KvKeep {
    uint8_t *pool;
    float *scales;
    const int *table;           // of the sequence, as it was
    const int *to;              // new pages, from the first that is built
    const int *index;
    size_t pool_layer, scales_layer;
    int first, kept, page0, pages;
    KvShape s;
};
constexpr int kKeepThreads = 256;

template <bool E4M3>
__global__ void __launch_bounds__(kKeepThreads) kv_keep_kernel(const __grid_constant__ KvKeep P) {
    extern __shared__ __align__(16) uint8_t keep_sm[];        // the page's codes
    __shared__ int source[128];                               // position of each token, -1 behind the last
    __shared__ float from_scale[128], top;
    const int h = blockIdx.y % P.s.kv_heads, layer = blockIdx.y / P.s.kv_heads, kv = blockIdx.z, D = P.s.head_dim, tid = threadIdx.x;
    const int shift = P.s.page_shift, tokens = 1 << shift, mask = tokens - 1;
    uint8_t *pool = P.pool + layer * P.pool_layer + h * kv_head_bytes(P.s) + kv * kv_half_bytes(P.s);
    float *scales = P.scales + layer * P.scales_layer + h * 2 + kv;
    const size_t page_bytes = kv_page_bytes(P.s);
    const int page_scales = P.s.kv_heads * 2;
#pragma unroll 1
    for (int i = blockIdx.x; i < P.pages; i += gridDim.x) {
        const int p0 = (P.page0 + i) << shift;
        if (tid < tokens) {
            const int pos = p0 + tid;
            const int src = pos < P.first ? pos : pos < P.first + P.kept ? P.first + P.index[pos - P.first] : -1;
            source[tid] = src;
            from_scale[tid] = src < 0 ? 0.0f : scales[static_cast<size_t>(P.table[src >> shift]) * page_scales];
        }
        __syncthreads();
        if (tid < 32) {
            float m = 0.0f;
            for (int t = tid; t < tokens; t += 32) m = fmaxf(m, from_scale[t]);
#pragma unroll
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (tid == 0) top = m;
        }
        __syncthreads();
        const float s1 = top;
        const int used = (min(P.first + P.kept - p0, tokens) + kKvSub - 1) / kKvSub;      // sub-blocks
        if (kv == 0) {
            const int per = D / 16;
            for (int j = tid; j < used * kKvSub * per; j += kKeepThreads) {
                const int t = j / per, k = (j - t * per) * 16, src = source[t];
                uint4 x = make_uint4(0, 0, 0, 0);
                uint8_t *c = reinterpret_cast<uint8_t *>(&x);
                if (src >= 0) {
                    const int o = src & mask;
                    x = *reinterpret_cast<const uint4 *>(pool + static_cast<size_t>(P.table[src >> shift]) * page_bytes + (o / kKvSub) * kv_sub_bytes(D) +
                                                         kv_k_offset(D, o % kKvSub, k));
                    const float s0 = from_scale[t];
                    if (s0 != s1) {
#pragma unroll
                        for (int b = 0; b < 16; ++b) c[b] = static_cast<uint8_t>(kv_recode<E4M3>(c[b], s0, s1));
                    }
                }
                *reinterpret_cast<uint4 *>(keep_sm + (t / kKvSub) * 16 * D + kv_k_offset(D, t % kKvSub, k)) = x;
            }
        } else {
            for (int j = tid; j < used * kKvSub * D; j += kKeepThreads) {
                const int sub = j / (kKvSub * D), in = j - sub * (kKvSub * D), v = in / 16, t = sub * kKvSub + kv_v_token(v, in % 16), src = source[t];
                int c = 0;
                if (src >= 0) {
                    const int o = src & mask;
                    c = pool[static_cast<size_t>(P.table[src >> shift]) * page_bytes + (o / kKvSub) * kv_sub_bytes(D) + kv_v_offset(o % kKvSub, kv_v_element(v, in % 16))];
                    const float s0 = from_scale[t];
                    if (s0 != s1) c = kv_recode<E4M3>(c, s0, s1);
                }
                keep_sm[j] = static_cast<uint8_t>(c);
            }
        }
        __syncthreads();
        const int page = P.to[i];
        for (int j = tid; j < used * D; j += kKeepThreads) {
            const int sub = j / D, v = j - sub * D;
            reinterpret_cast<uint4 *>(pool + static_cast<size_t>(page) * page_bytes + sub * kv_sub_bytes(D))[v] = reinterpret_cast<const uint4 *>(keep_sm + sub * 16 * D)[v];
        }
        if (tid == 0) scales[static_cast<size_t>(page) * page_scales] = s1;
        __syncthreads();
    }
}

}  // namespace wd
