// The 8-bit key/value cache: how a page lies in memory, how numbers become codes and codes numbers.
//
// pool    [layer][page][kv head][K: page_tokens D bytes | V: page_tokens D bytes]
// scales  [layer][page][kv head][2]  (F32; keys, values)
// reach   [layer][kv head]           how large and how small value scales have been since the cache began: largest exponent + 1024, 1024 - least exponent; 0: none
// book    int32 words: the step's header and entries, then the page table [max_seqs][max_pages]
//
// K and V are sub-blocks of 16 tokens, 16 D bytes each, laid out as the A operands of a matrix instruction of 16 x 8 x 16 want them: a lane
// (g = lane / 4, t = lane % 4) reads 16 bytes, a warp 512 bytes in a row.
//   K   rows are tokens:  [D / CW][16 tokens][CW], CW = 64 elements (32 where head_dim is no multiple of 64)
//   V   rows are elements of the head, the contraction runs over tokens: [D / 32][g][t][i][b] is element 8 i + g of the 32, token
//       2 t + (b & 1) + 8 (b >> 1)
// An int8 code c is held as the byte c + 128 (an f16 is made of it with one byte permutation and one subtraction), an e4m3 code as it is.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "wd_device.cuh"

namespace wd {

constexpr int kKvSub = 16;              // tokens of a sub-block
constexpr int kKvStepWords = 8;         // words of a step's entry: sequence, first row, rows, length with the step's tokens, first page item
constexpr int kKvHead = 8;              // words in front of the entries: sequences, rows, page items
constexpr float kKvLeastScale = 7.888609052210118e-31f;     // 2^-100: keeps 1 / scale and sums of it far inside F32

// Whether value scales may be so far apart that a weight times the one is nothing in F32 where that times the other is of size 1; and what stands for a
// scale of 0 (nothing but zeros): well below the others, so that its tokens cost no weight its place, and where they are not far apart no farther than that.
constexpr int kKvFar = 90;
__device__ __forceinline__ bool kv_far_apart(int2 reach) { return reach.x && (reach.x - 1024) - (1024 - reach.y) > kKvFar; }
__device__ __forceinline__ float kv_zero_scale(int2 reach) {
    const int hi = reach.x - 1024, lo = 1024 - reach.y;
    return reach.x == 0 || hi - lo > kKvFar ? kKvLeastScale : __uint_as_float(static_cast<uint32_t>(max(max(lo - 60, hi - kKvFar), -100) + 127) << 23);
}

enum : unsigned { kKvNonFinite = 32u };     // status bit: a NaN or an infinity was appended

struct KvShape {
    int heads, kv_heads, head_dim, page_shift, e4m3, max_pages;
};
__host__ __device__ inline int kv_cw(int d) { return d % 64 == 0 ? 64 : 32; }
__host__ __device__ inline size_t kv_sub_bytes(int d) { return static_cast<size_t>(d) * 16; }
__host__ __device__ inline size_t kv_half_bytes(const KvShape &s) { return static_cast<size_t>(s.head_dim) << s.page_shift; }       // keys or values of a page's head
__host__ __device__ inline size_t kv_head_bytes(const KvShape &s) { return 2 * kv_half_bytes(s); }
__host__ __device__ inline size_t kv_page_bytes(const KvShape &s) { return kv_head_bytes(s) * s.kv_heads; }
// offset in a sub-block of the 16 bytes of token t (0 .. 15) that hold the elements k .. k + 15 (k a multiple of 16) of a key
__host__ __device__ inline int kv_k_offset(int d, int t, int k) {
    const int cw = kv_cw(d);
    return (k / cw) * (16 * cw) + t * cw + k % cw;
}
// offset of one element of a value, and the token and element that byte j of the v-th 16 bytes stands for
__host__ __device__ inline int kv_v_offset(int t, int d) { return (d >> 5) * 512 + ((d & 7) * 4 + ((t & 7) >> 1)) * 16 + ((d & 31) >> 3) * 4 + (t & 1) + (t >> 3) * 2; }
__host__ __device__ inline int kv_v_token(int v, int j) { return (v & 3) * 2 + (j & 1) + ((j & 2) << 2); }
__host__ __device__ inline int kv_v_element(int v, int j) { return (v >> 5) * 32 + (j >> 2) * 8 + ((v & 31) >> 2); }

// ---- numbers of the rows ------------------------------------------------------------------------------------------------
enum { kRowsF32 = 0, kRowsF16 = 1, kRowsBF16 = 2 };
__device__ __forceinline__ void row_store(void *p, int type, size_t i, float v) {
    if (type == kRowsF32) static_cast<float *>(p)[i] = v;
    else if (type == kRowsF16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// 16 elements of a row, by reads of 16 bytes where `vec` says that they lie on such boundaries
template <class T>
__device__ __forceinline__ void row_load16(const T *p, bool vec, float *x) {
    if (vec) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; i += N) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p + i));
            const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
            for (int j = 0; j < N; ++j) x[i + j] = static_cast<float>(e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = static_cast<float>(p[i]);
    }
}
template <class T>
__device__ __forceinline__ T row_number(float v);
template <>
__device__ __forceinline__ float row_number<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half row_number<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 row_number<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ void row_pair(float *to, float a, float b) { to[0] = a, to[1] = b; }
__device__ __forceinline__ void row_pair(__half *to, float a, float b) { *reinterpret_cast<__half2 *>(to) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void row_pair(__nv_bfloat16 *to, float a, float b) { *reinterpret_cast<__nv_bfloat162 *>(to) = __floats2bfloat162_rn(a, b); }
// 8 x 8 matrix of 16-bit elements, a row's pairs in four lanes, turned
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// ---- codes --------------------------------------------------------------------------------------------------------------
// The code of the quotient n / s, to the nearest, ties to even, and exactly so: a quotient that F32 rounds onto the middle between two codes is
// told apart in 64 bits. (n = x, or an older code times its scale, has at most 32 significant bits and a middle at most 9, so that a quotient of
// 64 bits lies on a middle only where n / s does.)
__device__ __forceinline__ int e4m3_of(double q) {
    float f = __double2float_rz(q);
    if (static_cast<double>(f) != q) f = __uint_as_float(__float_as_uint(f) | 1u);        // to odd: the one rounding to come sees what was cut off
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(f));
    return r & 0xff;
}
template <bool E4M3>
__device__ __forceinline__ int kv_code_exact(double n, float s) {
    const double q = n / static_cast<double>(s);
    if (E4M3) return e4m3_of(q);
    return max(-127, min(127, __double2int_rn(q))) + 128;
}
// Four codes' values, and four quotients' codes. A quotient made as x * (1 / s), or as value * (s0 / s1), is off by at most 2^-22 of itself: `unsure` says that
// one of them is that near to a middle between codes (or is no number, or beyond the largest code), and then the codes are worked out by kv_code_exact.
// (int8: 2^23 + byte and 1.5 2^23 + quotient instead of conversions, which have a quarter of the rate.)
template <bool E4M3>
__device__ __forceinline__ void kv_values4(uint32_t w, float *v) {
    if (E4M3) {
        uint32_t lo, hi;
        asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
    }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t kv_codes4(const float *q, uint32_t &unsure) {
    if (E4M3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = __float_as_uint(q[i]) & 0x7fffffffu;
            // a middle; between 2^-11 and 2^-6 (codes without leading bit); over 448, or no number
            unsure |= (b & 0xfffffu) - 0x7fff0u <= 32u || b - 0x3a000000u < 0x2800000u || b > 0x43e00000u ? 1u << i : 0u;
        }
        uint32_t r;
        asm("{\n .reg .b16 a, b;\n cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n mov.b32 %0, {a, b};\n}" : "=r"(r) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]));
        return r;
    }
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t[i] = q[i] + 12583040.0f;
        unsure |= !(fabsf(q[i] - (t[i] - 12583040.0f)) <= 0.4999f) ? 1u << i : 0u;
    }
    return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
}
// the code of any x under s: an infinity becomes the largest code, a NaN zero; under a scale of 0 every code is zero (what reads the page counts on it)
template <bool E4M3>
__device__ __forceinline__ int kv_code_any(float x, float s) {
    if (s == 0.0f || x != x) return E4M3 ? 0 : 128;
    if (fabsf(x) > 3.402823466e38f) return E4M3 ? (x > 0.0f ? 0x7e : 0xfe) : (x > 0.0f ? 255 : 1);
    return kv_code_exact<E4M3>(static_cast<double>(x), s);
}
// 16 numbers -> codes under s, r = 1 / s (0 where s is: then every number is 0, or none)
template <bool E4M3>
__device__ __forceinline__ uint4 kv_encode16(const float *x, float s, float r) {
    uint32_t w[4], unsure = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q[4] = {x[4 * i] * r, x[4 * i + 1] * r, x[4 * i + 2] * r, x[4 * i + 3] * r};
        uint32_t some = 0;
        w[i] = kv_codes4<E4M3>(q, some);
        unsure |= some << (4 * i);
    }
    if (unsure) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (!(unsure >> i & 1u)) continue;
            const uint32_t c = static_cast<uint32_t>(kv_code_any<E4M3>(x[i], s)) << (8 * (i & 3));
            w[i / 4] = (w[i / 4] & ~(0xffu << (8 * (i & 3)))) | c;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// four codes under scale s0 as codes under s1 >= s0 (> 0), ratio = s0 / s1
template <bool E4M3>
__device__ __forceinline__ uint32_t kv_recode4(uint32_t w, float s0, float s1, float ratio) {
    float v[4];
    kv_values4<E4M3>(w, v);
    const float q[4] = {v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio};
    uint32_t unsure = 0, r = kv_codes4<E4M3>(q, unsure);
    if (unsure) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (unsure >> i & 1u)
                r = (r & ~(0xffu << (8 * i))) | static_cast<uint32_t>(kv_code_exact<E4M3>(static_cast<double>(v[i]) * static_cast<double>(s0), s1)) << (8 * i);
    }
    return r;
}
// four codes -> their values as f16 pairs (exact: both code sets are subsets of f16)
template <bool E4M3>
__device__ __forceinline__ void kv_halves(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (E4M3) {
        asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {        // 0x6400 | byte is 1024 + byte
        const __half2 off = __half2half2(__ushort_as_half(0x6480));
        uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), off), y = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    }
}

// the entry of the step that page item `item` belongs to: the last one whose items begin at or in front of it (all threads of the block)
__device__ __forceinline__ int kv_entry_of_item(const int *entries, int n, int item) {
    int at = -1;
    for (int i = 0; i < n; i += blockDim.x) {
        const int mine = i + static_cast<int>(threadIdx.x);
        at += __syncthreads_count(mine < n && entries[mine * kKvStepWords + 4] <= item);
    }
    return at;
}

}  // namespace wd
