// Kernels that keep the 8-bit cache: words of the book, numbers out (read), pages copied and tokens moved together (keep).
#pragma once

#include "wd_kv_layout.cuh"

namespace wd {

// ---- words of the book, by value: ordered by the stream, and no staging buffer that a later call could overwrite -----------------
template <int N>
struct KvWords {
    int n;
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

// ---- read -----------------------------------------------------------------------------------------------------------------
// Tokens first .. first + count - 1 of sequences as numbers, rows one after the other: [layer][row][kv head][D]. A block takes a sub-block of
// 16 tokens of a layer, all heads, keys and values; a warp 512 bytes, which are 16 tokens of 32 elements of a value's head (turned in shared
// memory, so that rows are written in pieces of 64 bytes and more). Bound: instruction issue (70 % of the slots).
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
    int n, vec;
    KvShape s;
    KvReadEntry e[kReadEntries];
};
constexpr int kReadThreads = 256;

template <class T, bool E4M3>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const __grid_constant__ KvRead P) {
    constexpr int PITCH = 32 + 16 / sizeof(T);
    __shared__ __align__(16) T turned[kReadThreads / 32][kKvSub][PITCH];
    const int item = blockIdx.x, layer = blockIdx.y, D = P.s.head_dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
    const uint8_t *base = P.pool + layer * P.pool_layer + static_cast<size_t>(page) * kv_page_bytes(P.s) + ((t0 & ((1 << shift) - 1)) / kKvSub) * kv_sub_bytes(D);
    const float *scales = P.scales + layer * P.scales_layer + static_cast<size_t>(page) * P.s.kv_heads * 2;
    const size_t pitch = static_cast<size_t>(P.s.kv_heads) * D, head_bytes = kv_head_bytes(P.s), half = kv_half_bytes(P.s);
    T *ko = static_cast<T *>(P.out[0]), *vo = static_cast<T *>(P.out[1]);
    const size_t row0 = static_cast<size_t>(e.row0 + t0 - e.first);        // of token 0, which may lie in front of the rows
    const int per_head = D / 32, units = P.s.kv_heads * per_head, cw = kv_cw(D);         // a unit is 512 bytes
    constexpr int N = 16 / sizeof(T);
#pragma unroll 2
    for (int u = warp; u < 2 * units; u += kReadThreads / 32) {
        const int kv = u >= units, in = u - kv * units, h = in / per_head, blk = in - h * per_head;
        if ((kv ? vo : ko) == nullptr) continue;
        const uint4 x = *reinterpret_cast<const uint4 *>(base + h * head_bytes + kv * half + blk * 512 + lane * 16);
        const float s = scales[h * 2 + kv];
        float v[16];
        kv_values4<E4M3>(x.x, v), kv_values4<E4M3>(x.y, v + 4), kv_values4<E4M3>(x.z, v + 8), kv_values4<E4M3>(x.w, v + 12);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __fmul_rn(v[j], s);
        if (kv == 0) {
            const int at = blk * 512 + lane * 16, token = at % (16 * cw) / cw, k = at / (16 * cw) * cw + at % cw;
            if (token >= a && token < b) {
                T *to = ko + layer * P.out_layer + (row0 + token) * pitch + static_cast<size_t>(h) * D + k;
                __align__(16) T y[16];
#pragma unroll
                for (int j = 0; j < 16; j += 2) row_pair(y + j, v[j], v[j + 1]);
                if (P.vec) {
#pragma unroll
                    for (int j = 0; j < 16; j += N) *reinterpret_cast<uint4 *>(to + j) = *reinterpret_cast<const uint4 *>(y + j);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) to[j] = y[j];
                }
            }
        } else {
            __syncwarp();
            if constexpr (sizeof(T) == 2) {
                // word i: element 8 i + g of tokens 2 t, 2 t + 1 and 8 more; turned, a lane has elements 8 i + 2 t and the next of tokens g and g + 8
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    __align__(4) T pair[4];
                    row_pair(pair, v[4 * i], v[4 * i + 1]);
                    row_pair(pair + 2, v[4 * i + 2], v[4 * i + 3]);
                    const uint32_t *w = reinterpret_cast<const uint32_t *>(pair);
                    *reinterpret_cast<uint32_t *>(&turned[warp][lane >> 2][8 * i + 2 * (lane & 3)]) = transposed(w[0]);
                    *reinterpret_cast<uint32_t *>(&turned[warp][(lane >> 2) + 8][8 * i + 2 * (lane & 3)]) = transposed(w[1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) turned[warp][kv_v_token(lane, j)][kv_v_element(lane, j)] = row_number<T>(v[j]);
            }
            __syncwarp();
            T *to = vo + layer * P.out_layer + row0 * pitch + static_cast<size_t>(h) * D + blk * 32;
            if (P.vec) {
#pragma unroll
                for (int i = lane; i < kKvSub * 32 / N; i += 32) {
                    const int token = i / (32 / N), d = i % (32 / N) * N;
                    if (token >= a && token < b) *reinterpret_cast<uint4 *>(to + token * pitch + d) = *reinterpret_cast<const uint4 *>(&turned[warp][token][d]);
                }
            } else {
                for (int token = a; token < b; ++token) to[token * pitch + lane] = turned[warp][token][lane];
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
    int page_scales;
    int2 pair[kCopyPairs];      // from, to; a block of the second index each (the third: layers)
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
// its tokens come from pages behind it (or itself), its scale is the largest of theirs, codes of smaller ones are rounded anew. Where there are no free
// pages to be had, a block walks over the pages in their order, reading all of a page's tokens before it writes (the order is the bound: the first call on a
// cache that keeps 3,301 of 5,900 tokens in 16 layers of 8 heads of 64 takes 220 us, into new pages 127).
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
// byte shift8 / 8 of each word as the bytes of one, and the bytes of z as byte q of each word
__device__ __forceinline__ uint32_t kv_byte_of_each(const uint4 &y, int shift8) {
    return __byte_perm(__byte_perm(y.x >> shift8, y.y >> shift8, 0x0040), __byte_perm(y.z >> shift8, y.w >> shift8, 0x0040), 0x5410);
}
__device__ __forceinline__ void kv_byte_to_each(uint4 &x, uint32_t z, int q) {
    const uint32_t shift = 8 * q;
    x.x |= (z & 0xffu) << shift, x.y |= (z >> 8 & 0xffu) << shift, x.z |= (z >> 16 & 0xffu) << shift, x.w |= (z >> 24) << shift;
}

template <bool E4M3>
__global__ void __launch_bounds__(kKeepThreads) kv_keep_kernel(const __grid_constant__ KvKeep P) {
    extern __shared__ __align__(16) uint8_t keep_sm[];        // the page's codes
    __shared__ int source[128];                               // position of each token, -1 behind the last
    __shared__ float from_scale[128], top;
    __shared__ size_t from_page[128];
    const int h = blockIdx.y % P.s.kv_heads, layer = blockIdx.y / P.s.kv_heads, kv = blockIdx.z, D = P.s.head_dim, tid = threadIdx.x;
    const int shift = P.s.page_shift, tokens = 1 << shift, mask = tokens - 1;
    uint8_t *pool = P.pool + layer * P.pool_layer + h * kv_head_bytes(P.s) + kv * kv_half_bytes(P.s);
    float *scales = P.scales + layer * P.scales_layer + h * 2 + kv;
    const size_t page_bytes = kv_page_bytes(P.s);
    const int page_scales = P.s.kv_heads * 2;
#pragma unroll 1
    for (int i = 0; i < P.pages; ++i) {
        const int p0 = (P.page0 + i) << shift;
        if (tid < tokens) {
            const int pos = p0 + tid;
            const int src = pos < P.first ? pos : pos < P.first + P.kept ? P.first + P.index[pos - P.first] : -1;
            source[tid] = src;
            const size_t page = src < 0 ? 0 : static_cast<size_t>(P.table[src >> shift]);
            from_page[tid] = page * page_bytes;
            from_scale[tid] = src < 0 ? 0.0f : scales[page * page_scales];
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
        for (int j = tid; j < used * D; j += kKeepThreads) {         // 16 bytes each
            const int sub = j / D, v = j - sub * D;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (kv == 0) {
                const int cw = kv_cw(D), at = v * 16, t = sub * kKvSub + at % (16 * cw) / cw, src = source[t];
                if (src >= 0) {
                    const int o = src & mask;
                    x = *reinterpret_cast<const uint4 *>(pool + from_page[t] + (o / kKvSub) * kv_sub_bytes(D) + (o % kKvSub) * cw + at / (16 * cw) * (16 * cw) + at % cw);
                    const float s0 = from_scale[t];
                    if (s0 != s1) {
                        const float ratio = __fdiv_rn(s0, s1);
                        x = make_uint4(kv_recode4<E4M3>(x.x, s0, s1, ratio), kv_recode4<E4M3>(x.y, s0, s1, ratio), kv_recode4<E4M3>(x.z, s0, s1, ratio), kv_recode4<E4M3>(x.w, s0, s1, ratio));
                    }
                }
            } else {
                // four tokens; of each one the four elements are at one place of the words of 16 bytes
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int t = sub * kKvSub + kv_v_token(v, q), src = source[t];
                    if (src < 0) continue;
                    const int o = src & mask;
                    const uint8_t *p = pool + from_page[t] + (o / kKvSub) * kv_sub_bytes(D) + kv_v_offset(o % kKvSub, kv_v_element(v, 0));
                    const uint4 y = *reinterpret_cast<const uint4 *>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
                    const int shift8 = 8 * static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
                    uint32_t z = kv_byte_of_each(y, shift8);
                    const float s0 = from_scale[t];
                    if (s0 != s1) z = kv_recode4<E4M3>(z, s0, s1, __fdiv_rn(s0, s1));
                    kv_byte_to_each(x, z, q);
                }
            }
            reinterpret_cast<uint4 *>(keep_sm)[j] = x;
        }
        __syncthreads();
        const int page = P.to[i];
        for (int j = tid; j < used * D; j += kKeepThreads) {
            const int sub = j / D, v = j - sub * D;
            reinterpret_cast<uint4 *>(pool + static_cast<size_t>(page) * page_bytes + sub * kv_sub_bytes(D))[v] = reinterpret_cast<const uint4 *>(keep_sm)[j];
        }
        if (tid == 0) scales[static_cast<size_t>(page) * page_scales] = s1;
        __syncthreads();
    }
}

// The same into new pages, which need no order: a block builds a page of a layer for up to eight heads, keys and values, and writes what it gathers. (With a
// block for each head, the chain of index, table and scale in front of the first code was most of its time: 3,301 of 5,900 tokens in 16 layers of 8 heads
// of 64, 92 us; so 73, and 20 less since the tokens' places are worked out once for all heads. Bound: instruction issue, 62 % of the slots then; its 110 MB
// would take 17 us.)
constexpr int kKeepHeads = 8;
template <bool E4M3>
__global__ void __launch_bounds__(kKeepThreads) kv_keep_new_kernel(const __grid_constant__ KvKeep P) {
    __shared__ int source[128];                               // position of each token, -1 behind the last
    __shared__ size_t from_page[128];
    __shared__ float from_scale[2 * kKeepHeads][128], top[2 * kKeepHeads];
    const int i = blockIdx.x, layer = blockIdx.y, h0 = blockIdx.z * kKeepHeads, hk_n = 2 * min(kKeepHeads, P.s.kv_heads - h0), D = P.s.head_dim, tid = threadIdx.x;
    const int lane = tid & 31, shift = P.s.page_shift, tokens = 1 << shift, mask = tokens - 1, page_scales = P.s.kv_heads * 2;
    uint8_t *pool = P.pool + layer * P.pool_layer + h0 * kv_head_bytes(P.s);
    float *scales = P.scales + layer * P.scales_layer + h0 * 2;
    const size_t page_bytes = kv_page_bytes(P.s), half = kv_half_bytes(P.s);
    const int p0 = (P.page0 + i) << shift;
    if (tid < tokens) {
        const int pos = p0 + tid, src = pos < P.first ? pos : pos < P.first + P.kept ? P.first + P.index[pos - P.first] : -1;
        source[tid] = src;
        from_page[tid] = src < 0 ? 0 : static_cast<size_t>(P.table[src >> shift]);
    }
    __syncthreads();
#pragma unroll 4
    for (int u = tid; u < tokens * hk_n; u += kKeepThreads) {
        const int t = u & mask, hk = u >> shift;
        from_scale[hk][t] = source[t] < 0 ? 0.0f : scales[from_page[t] * page_scales + hk];
    }
    __syncthreads();
    for (int hk = tid >> 5; hk < hk_n; hk += kKeepThreads / 32) {
        float m = 0.0f;
        for (int t = lane; t < tokens; t += 32) m = fmaxf(m, from_scale[hk][t]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) top[hk] = m;
    }
    __syncthreads();
    const size_t page = static_cast<size_t>(P.to[i]);
    const int used = (min(P.first + P.kept - p0, tokens) + kKvSub - 1) / kKvSub, vecs = used * D, cw = kv_cw(D);
    // 16 bytes of each head: where they come from and go to is the same for all of them
    const size_t head_bytes = kv_head_bytes(P.s);
#pragma unroll 1
    for (int j = tid; j < vecs; j += kKeepThreads) {
        const int sub = j / D, v = j - sub * D;
        uint8_t *to = pool + page * page_bytes + sub * kv_sub_bytes(D) + v * 16;
        {
            const int at = v * 16, t = sub * kKvSub + at % (16 * cw) / cw, src = source[t], o = max(src, 0) & mask;
            const uint8_t *from = pool + from_page[t] * page_bytes + (o / kKvSub) * kv_sub_bytes(D) + (o % kKvSub) * cw + at / (16 * cw) * (16 * cw) + at % cw;
#pragma unroll 4
            for (int hk = 0; hk < hk_n; hk += 2) {
                uint4 x = *reinterpret_cast<const uint4 *>(from + (hk >> 1) * head_bytes);
                const float s0 = from_scale[hk][t], s1 = top[hk];
                if (s0 != s1 && s0 > 0.0f) {        // (a scale of 0: codes of 0 under any scale)
                    const float ratio = __fdiv_rn(s0, s1);
                    x = make_uint4(kv_recode4<E4M3>(x.x, s0, s1, ratio), kv_recode4<E4M3>(x.y, s0, s1, ratio), kv_recode4<E4M3>(x.z, s0, s1, ratio), kv_recode4<E4M3>(x.w, s0, s1, ratio));
                }
                *reinterpret_cast<uint4 *>(to + (hk >> 1) * head_bytes) = x;           // (behind the last token: codes of some other one)
            }
        }
        int t[4], shift8[4];
        const uint8_t *from[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            t[q] = sub * kKvSub + kv_v_token(v, q);
            const int o = max(source[t[q]], 0) & mask;
            const uint8_t *p = pool + from_page[t[q]] * page_bytes + half + (o / kKvSub) * kv_sub_bytes(D) + kv_v_offset(o % kKvSub, kv_v_element(v, 0));
            from[q] = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
            shift8[q] = 8 * static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
        }
#pragma unroll 2
        for (int hk = 1; hk < hk_n; hk += 2) {
            uint4 y[4], x = make_uint4(0, 0, 0, 0);
            const float s1 = top[hk];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = *reinterpret_cast<const uint4 *>(from[q] + (hk >> 1) * head_bytes);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t z = kv_byte_of_each(y[q], shift8[q]);
                const float s0 = from_scale[hk][t[q]];
                if (s0 != s1 && s0 > 0.0f) z = kv_recode4<E4M3>(z, s0, s1, __fdiv_rn(s0, s1));
                kv_byte_to_each(x, z, q);
            }
            *reinterpret_cast<uint4 *>(to + half + (hk >> 1) * head_bytes) = x;
        }
    }
    if (tid < hk_n) scales[page * page_scales + tid] = top[tid];
}

}  // namespace wd
