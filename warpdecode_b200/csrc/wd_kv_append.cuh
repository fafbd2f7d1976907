// Rows of a step into the 8-bit cache (append).
#pragma once

#include "wd_kv_layout.cuh"

namespace wd {

// A block takes the step's tokens that lie in one page, one kv head, keys (blockIdx.z = 0) or values. Two passes over its rows: the largest
// magnitude, from which the scale follows, then the codes (the rows come from the caches the second time). A page that held tokens before keeps its
// scale unless the new ones need a larger one; then the codes that are there are rounded anew. Values are turned in shared memory.
// Bound: instruction issue for a prompt (8,191 tokens of 8 heads of 128, written and read back: 52 us, 1.9 TB/s over both), the chain entry -> table ->
// scale -> rows for one token of each of 64 sequences (with the reading back 18.5 us).
struct KvAppend {
    uint8_t *pool;              // of the layer
    float *scales;              // of the layer
    int2 *reach;                // of the layer
    const int *book;
    const int *table;
    const void *rows[2];
    long long stride[2];
    unsigned *status;
    int vec[2];                 // rows lie on boundaries of 16 bytes
    KvShape s;
};

// Where a page item of the step lies: the step's tokens a .. b - 1 of a page.
struct KvPagePart {
    int row, page, a, b, place; // row: of the step, of token a; place: of token a in its sequence
};
// (all threads of the block)
__device__ __forceinline__ KvPagePart kv_page_part(const int *book, const int *table, const KvShape &s, int n_seq, int item) {
    const int *entries = book + kKvHead;
    const int *e = entries + kv_entry_of_item(entries, n_seq, item) * kKvStepWords;
    const int4 e0 = *reinterpret_cast<const int4 *>(e);
    const int seq = e0.x, row0 = e0.y, count = e0.z, length = e0.w, begin = length - count;
    const int logical = (begin >> s.page_shift) + item - e[4], page0 = logical << s.page_shift;
    KvPagePart r;
    r.a = max(begin - page0, 0);
    r.b = min(length - page0, 1 << s.page_shift);
    r.page = table[static_cast<size_t>(seq) * s.max_pages + logical];
    r.row = row0 + page0 + r.a - begin;
    r.place = page0 + r.a;
    return r;
}

// The part's codes of head h (kv = 0: keys, 1: values), and how they are made: all threads of the block, one after the other
//   top     the largest finite magnitude of what load(t, k, x) gives, 16 numbers from element k on of the part's tokens 0 .. n - 1, and whether there is one that is not finite
//   scale   the page's scale, and the codes of the tokens in front under it where it has grown
//   codes   of the part's tokens t0 .. t0 + n - 1, which load() counts from 0 (values: all of them at once)
struct KvPartScale {
    float s, r;                 // r = 1 / s, 0 where s is
};
template <int THREADS, class Load>
__device__ __forceinline__ float kv_part_top(int D, int n, Load load, float top, int &bad) {
    const int per = D / 16, groups = n * per;
    for (int i = threadIdx.x; i < groups; i += THREADS) {
        const int t = i / per, k = (i - t * per) * 16;
        float x[16];
        load(t, k, x);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float y = fabsf(x[j]);
            if (y <= 3.402823466e38f) top = fmaxf(top, y);
            else bad = 1;
        }
    }
    return top;
}
template <bool E4M3, int THREADS>
__device__ __forceinline__ KvPartScale kv_part_scale(const KvAppend &P, const KvPagePart &at, int h, int kv, float top, int bad, float *part, int &bad_any) {
    const int tid = threadIdx.x, D = P.s.head_dim, a = at.a;
    uint8_t *base = P.pool + static_cast<size_t>(at.page) * kv_page_bytes(P.s) + h * kv_head_bytes(P.s) + kv * kv_half_bytes(P.s);
    const float *scale = P.scales + (static_cast<size_t>(at.page) * P.s.kv_heads + h) * 2 + kv;
    const float s0 = a > 0 ? *scale : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (tid == 0) bad_any = 0;
    __syncthreads();
    if ((tid & 31) == 0) part[tid >> 5] = top;
    if (bad) bad_any = 1;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, part[w]);
    if (tid == 0 && bad_any) atomicOr(P.status, kKvNonFinite);
    const float need = top > 0.0f ? fmaxf(__fdiv_rn(top, E4M3 ? 448.0f : 127.0f), kKvLeastScale) : 0.0f;
    const float s1 = fmaxf(s0, need), r = s1 > 0.0f ? __fdiv_rn(1.0f, s1) : 0.0f;
    if (a > 0 && s1 != s0) {        // the codes of the tokens 0 .. a - 1 under the larger scale
        const int vecs = ((a + kKvSub - 1) / kKvSub) * D;
        const float ratio = __fdiv_rn(s0, s1);
        for (int i = tid; i < vecs; i += THREADS) {
            const int sub = i / D, v = i - sub * D, cw = kv_cw(D), token = (v * 16 % (16 * cw)) / cw;      // (of keys)
            if (kv == 0 && sub * kKvSub + token >= a) continue;        // another thread may have written its new codes already
            uint4 *p = reinterpret_cast<uint4 *>(base + sub * kv_sub_bytes(D)) + v;
            const uint4 x = *p;
            uint4 y = make_uint4(kv_recode4<E4M3>(x.x, s0, s1, ratio), kv_recode4<E4M3>(x.y, s0, s1, ratio), kv_recode4<E4M3>(x.z, s0, s1, ratio), kv_recode4<E4M3>(x.w, s0, s1, ratio));
            if (kv) {               // tokens from a on are written behind
                uint32_t mask = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) mask |= sub * kKvSub + kv_v_token(v, j) < a ? 0xffu << (8 * j) : 0u;
                y = make_uint4((y.x & mask) | (x.x & ~mask), (y.y & mask) | (x.y & ~mask), (y.z & mask) | (x.z & ~mask), (y.w & mask) | (x.w & ~mask));
            }
            *p = y;
        }
    }
    return {s1, r};
}
template <bool E4M3, int THREADS, class Load>
__device__ __forceinline__ void kv_part_codes(const KvAppend &P, const KvPagePart &at, int h, int kv, KvPartScale sc, uint8_t *app_sm, int t0, int n, Load load) {
    const int tid = threadIdx.x, D = P.s.head_dim, a = at.a, b = at.b, per = D / 16, groups = n * per, sub0 = a / kKvSub;
    uint8_t *base = P.pool + static_cast<size_t>(at.page) * kv_page_bytes(P.s) + h * kv_head_bytes(P.s) + kv * kv_half_bytes(P.s);
    for (int i = tid; i < groups; i += THREADS) {
        const int t = i / per, k = (i - t * per) * 16, token = a + t0 + t;
        float y[16];
        load(t, k, y);
        const uint4 x = kv_encode16<E4M3>(y, sc.s, sc.r);
        const uint8_t *c = reinterpret_cast<const uint8_t *>(&x);
        if (kv == 0) {
            *reinterpret_cast<uint4 *>(base + (token / kKvSub) * kv_sub_bytes(D) + kv_k_offset(D, token % kKvSub, k)) = x;
        } else {
            uint8_t *to = app_sm + (token / kKvSub - sub0) * 16 * D + kv_v_offset(token % kKvSub, k);
#pragma unroll
            for (int j = 0; j < 16; ++j) to[(j & 7) * 64 + (j >> 3) * 4] = c[j];       // element k + j: k is a multiple of 16, so that only j moves the byte
        }
    }
    __syncthreads();        // the turned codes are there, and the older ones that share 16 bytes with them
    if (kv == 1) {
        const int vecs = ((b - 1) / kKvSub + 1 - sub0) * D;
        for (int i = tid; i < vecs; i += THREADS) {
            const int sub = sub0 + i / D, v = i % D, lo = a - sub * kKvSub, hi = b - sub * kKvSub;
            uint8_t *to = base + sub * kv_sub_bytes(D) + v * 16;
            const uint4 x = reinterpret_cast<const uint4 *>(app_sm)[i];
            const uint8_t *c = reinterpret_cast<const uint8_t *>(&x);
            if (lo <= 0 && hi >= kKvSub) {
                *reinterpret_cast<uint4 *>(to) = x;
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (kv_v_token(v, j) >= lo && kv_v_token(v, j) < hi) to[j] = c[j];
            }
        }
    }
}
// the scale into the page; `reach` as the layer's was before (of values)
__device__ __forceinline__ void kv_part_end(const KvAppend &P, const KvPagePart &at, int h, int kv, float s1, int2 reach) {
    if (threadIdx.x != 0) return;
    P.scales[(static_cast<size_t>(at.page) * P.s.kv_heads + h) * 2 + kv] = s1;
    const int at_1 = static_cast<int>(__float_as_uint(s1) >> 23) - 127;
    if (kv && s1 > 0.0f && (at_1 + 1024 > reach.x || 1024 - at_1 > reach.y)) {
        atomicMax(&P.reach[h].x, at_1 + 1024);
        atomicMax(&P.reach[h].y, 1024 - at_1);
    }
}
// All of it, for rows in memory.
template <class T, bool E4M3, int THREADS>
__device__ __forceinline__ void kv_append_part(const KvAppend &P, const KvPagePart &at, int h, int kv, uint8_t *app_sm, float *part, int &bad_any) {
    const size_t stride = static_cast<size_t>(P.stride[kv]);
    const bool vec = P.vec[kv] != 0;
    const T *rows = static_cast<const T *>(P.rows[kv]) + static_cast<size_t>(at.row) * stride + static_cast<size_t>(h) * P.s.head_dim;
    const int2 reach = threadIdx.x == 0 && kv ? P.reach[h] : make_int2(0, 0);        // (as it was, or newer)
    auto load = [&](int t, int k, float *x) { row_load16(rows + t * stride + k, vec, x); };
    int bad = 0;
    const float top = kv_part_top<THREADS>(P.s.head_dim, at.b - at.a, load, 0.0f, bad);
    const KvPartScale sc = kv_part_scale<E4M3, THREADS>(P, at, h, kv, top, bad, part, bad_any);
    kv_part_codes<E4M3, THREADS>(P, at, h, kv, sc, app_sm, 0, at.b - at.a, load);
    kv_part_end(P, at, h, kv, sc.s, reach);
}

template <class T, bool E4M3, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 4 : 16) kv_append_kernel(const __grid_constant__ KvAppend P) {
    extern __shared__ __align__(16) uint8_t app_sm[];           // values: the codes of the sub-blocks that the rows touch
    __shared__ float part[THREADS / 32];
    __shared__ int bad_any;
    const int n_seq = P.book[0], n_items = P.book[2];
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const KvPagePart at = kv_page_part(P.book, P.table, P.s, n_seq, item);
        kv_append_part<T, E4M3, THREADS>(P, at, blockIdx.y, blockIdx.z, app_sm, part, bad_any);
        __syncthreads();
    }
}

}  // namespace wd
