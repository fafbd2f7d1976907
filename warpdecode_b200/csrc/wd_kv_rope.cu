// Norms and rotary positions of a step's queries and keys, the keys and values into the 8-bit cache on the way (wd_rope_*, wd_kv_append_rope).
//
//   n = x w / sqrt(mean x^2 + eps);   pair p of a head: angle a = position f_p,  (y0, y1) = factor (n0 cos a - n1 sin a, n1 cos a + n0 sin a)
//
// A block takes the step's tokens that lie in one page and one kv head: its keys (blockIdx.z = 0), its values (1), or some of the query heads that share it
// (2 and up). An angle is made once for all of a block's query heads of a token.
//
// Angles are made in turns, position (f_p / 2 pi) in 64 bits less the nearest whole number: in 32 bits the position 131,072 is off by 2^-8 radians. Queries
// are rotated in F32, by the sine of that rest rounded to F32 (off by 2^-26 of a turn at most: 1e-7 of an element). Keys in 64 bits, rounded to F32 once: then the code is the same however the sums are ordered, but for one number in 2^25, and the same
// rows again leave the cache as it is. The rotated keys of a page wait in shared memory for the page's scale, as many tokens at a time as it holds; those
// of a page that has more are made a second time.
//
// Few tokens are a chain of latencies (64 sequences, a token each, 32/8 heads of 128: 10.6 us). Many are bound by instruction issue and conversions of 64 bits, at two blocks an SM:
// 4,000 tokens of 32/8 heads of 64 29 us (57 MB, 8.8 at the memory's rate), 5,003 of 128 by three axes 76, of which the codes of keys and values are 26, the keys' rotation 14 and
// the queries 34. Every kv head's blocks make the step's angles anew, in each layer.
#include <cmath>
#include <memory>

#include "wd_kv_append.cuh"
#include "wd_kv_host.h"

using namespace wd_kv;

struct wd_rope {
    wd_rope_config cfg{};
    int section_end[4] = {};
    double turns[128] = {};         // of each pair, for a step of one in its position
};

namespace wd {
namespace {

constexpr int kRopePairs = 4;       // of a lane: heads of up to 256
constexpr int kRopeHeld = 16384;    // floats of rotated keys that a block holds at most; the codes of a page's values are no more bytes than these

struct KvRope {
    KvAppend a;
    const void *q;
    void *q_out;
    long long q_stride, q_out_stride;
    const int *positions;           // null: the tokens' own places
    const float *q_norm, *k_norm;
    float eps, factor;
    int rotary, neighbours, n_axes, q_parts, held;      // held: tokens that shared memory has room for
    int section_end[4];
    double turns[128];
};

// The pairs of a lane: their elements, axis and frequency. Pairs behind the rotated ones are two elements that are only brought through.
struct RopeLane {
    int e0[kRopePairs], e1[kRopePairs], axis[kRopePairs];
    double turns[kRopePairs];
    bool is[kRopePairs], turned[kRopePairs];
};
__device__ __forceinline__ RopeLane rope_lane(const KvRope &P, int lane) {
    RopeLane r;
#pragma unroll
    for (int i = 0; i < kRopePairs; ++i) {
        const int p = lane + 32 * i, half = P.rotary / 2;
        r.is[i] = p < P.a.s.head_dim / 2;
        r.turned[i] = p < half;
        r.e0[i] = r.turned[i] && !P.neighbours ? p : 2 * p;
        r.e1[i] = r.turned[i] && !P.neighbours ? p + half : 2 * p + 1;
        r.axis[i] = (p >= P.section_end[0]) + (p >= P.section_end[1]) + (p >= P.section_end[2]);
        r.turns[i] = r.turned[i] ? P.turns[p] : 0.0;
    }
    return r;
}
// 2 (turns less the nearest whole number): what the functions of pi times x take
__device__ __forceinline__ double rope_angle(const KvRope &P, const RopeLane &l, int i, int row, int place) {
    const double a = static_cast<double>(P.positions ? P.positions[static_cast<size_t>(row) * P.n_axes + min(l.axis[i], P.n_axes - 1)] : place) * l.turns[i];
    return 2.0 * (a - rint(a));
}

// where a float of the held rows is: 16 of them that one thread reads lie in other banks than its neighbours'
__device__ __forceinline__ int rope_held(int e) { return (e & ~15) | ((((e >> 2) + (e >> 5)) & 3) << 2) | (e & 3); }

// ---- few tokens, or rows that do not lie on boundaries of 16 bytes: a warp a token's head, a lane the pairs lane, lane + 32, ... ----------------
template <class T, bool E4M3, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_rope_kernel(const __grid_constant__ KvRope P) {
    extern __shared__ __align__(16) uint8_t rope_sm[];           // keys: rotated rows; values: the codes of the sub-blocks that the rows touch
    __shared__ float part[THREADS / 32];
    __shared__ int bad_any;
    constexpr int W = THREADS / 32;
    const int n_seq = P.a.book[0], n_items = P.a.book[2], h = blockIdx.y, D = P.a.s.head_dim, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const KvPagePart at = kv_page_part(P.a.book, P.a.table, P.a.s, n_seq, item);
        const int n = at.b - at.a;
        if (blockIdx.z == 1) {
            kv_append_part<T, E4M3, THREADS>(P.a, at, h, 1, rope_sm, part, bad_any);
        } else if (blockIdx.z == 0) {
            const RopeLane l = rope_lane(P, lane);
            const T *rows = static_cast<const T *>(P.a.rows[0]) + static_cast<size_t>(at.row) * P.a.stride[0] + static_cast<size_t>(h) * D;
            float *held = reinterpret_cast<float *>(rope_sm);
            auto rotate = [&](int t0, int m) {
                for (int t = warp; t < m; t += W) {
                    const T *x = rows + static_cast<size_t>(t0 + t) * P.a.stride[0];
                    float x0[kRopePairs], x1[kRopePairs];
#pragma unroll
                    for (int i = 0; i < kRopePairs; ++i) {
                        x0[i] = l.is[i] ? static_cast<float>(x[l.e0[i]]) : 0.0f;
                        x1[i] = l.is[i] ? static_cast<float>(x[l.e1[i]]) : 0.0f;
                    }
                    double inv = 1.0;
                    if (P.k_norm) {
                        double sum = 0.0;
#pragma unroll
                        for (int i = 0; i < kRopePairs; ++i) sum += static_cast<double>(x0[i]) * x0[i] + static_cast<double>(x1[i]) * x1[i];
#pragma unroll
                        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        inv = 1.0 / sqrt(sum / D + static_cast<double>(P.eps));
                    }
#pragma unroll
                    for (int i = 0; i < kRopePairs; ++i) {
                        if (!l.is[i]) continue;
                        double n0 = x0[i], n1 = x1[i];
                        if (P.k_norm) n0 = n0 * inv * P.k_norm[l.e0[i]], n1 = n1 * inv * P.k_norm[l.e1[i]];
                        if (l.turned[i]) {
                            double sn, cs;
                            sincospi(rope_angle(P, l, i, at.row + t0 + t, at.place + t0 + t), &sn, &cs);
                            const double f = P.factor, y0 = f * (n0 * cs - n1 * sn), y1 = f * (n1 * cs + n0 * sn);
                            n0 = y0, n1 = y1;
                        }
                        held[rope_held(t * D + l.e0[i])] = static_cast<float>(n0);
                        held[rope_held(t * D + l.e1[i])] = static_cast<float>(n1);
                    }
                }
            };
            auto load = [&](int t, int k, float *x) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 v = *reinterpret_cast<const float4 *>(held + rope_held(t * D + k + 4 * j));
                    x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
                }
            };
            float top = 0.0f;
            int bad = 0;
            for (int t0 = 0; t0 < n; t0 += P.held) {
                if (t0 > 0) __syncthreads();
                rotate(t0, min(P.held, n - t0));
                __syncthreads();
                top = kv_part_top<THREADS>(D, min(P.held, n - t0), load, top, bad);
            }
            const KvPartScale sc = kv_part_scale<E4M3, THREADS>(P.a, at, h, 0, top, bad, part, bad_any);
            for (int t0 = 0; t0 < n; t0 += P.held) {
                if (n > P.held) {
                    __syncthreads();
                    rotate(t0, min(P.held, n - t0));
                    __syncthreads();
                }
                kv_part_codes<E4M3, THREADS>(P.a, at, h, 0, sc, nullptr, t0, min(P.held, n - t0), load);
            }
            kv_part_end(P.a, at, h, 0, sc.s, make_int2(0, 0));
        } else {
            const RopeLane l = rope_lane(P, lane);
            const int g = P.a.s.heads / P.a.s.kv_heads, part_q = blockIdx.z - 2, h0 = h * g + g * part_q / P.q_parts, h1 = h * g + g * (part_q + 1) / P.q_parts;
            // a warp a token; where there are fewer tokens, some warps share one's heads
            const int share = n < W ? W / n : 1;
            for (int t = warp / share; t < n; t += W / share) {
                float cs[kRopePairs], sn[kRopePairs];
#pragma unroll
                for (int i = 0; i < kRopePairs; ++i) {
                    cs[i] = 1.0f, sn[i] = 0.0f;
                    if (!l.turned[i]) continue;
                    sincospif(static_cast<float>(rope_angle(P, l, i, at.row + t, at.place + t)), &sn[i], &cs[i]);
                    cs[i] *= P.factor, sn[i] *= P.factor;
                }
                const T *from = static_cast<const T *>(P.q) + static_cast<size_t>(at.row + t) * P.q_stride;
                T *to = static_cast<T *>(P.q_out) + static_cast<size_t>(at.row + t) * P.q_out_stride;
                for (int head = h0 + warp % share; head < h1; head += share) {
                    const T *x = from + static_cast<size_t>(head) * D;
                    T *y = to + static_cast<size_t>(head) * D;
                    float x0[kRopePairs], x1[kRopePairs];
#pragma unroll
                    for (int i = 0; i < kRopePairs; ++i) {
                        x0[i] = l.is[i] ? static_cast<float>(x[l.e0[i]]) : 0.0f;
                        x1[i] = l.is[i] ? static_cast<float>(x[l.e1[i]]) : 0.0f;
                    }
                    if (P.q_norm) {
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < kRopePairs; ++i) sum = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], sum));
#pragma unroll
                        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        float inv = __frsqrt_rn(sum / D + P.eps);
                        if (!(sum > 1e-30f && sum < 1e38f)) {           // squares that F32 does not hold
                            double wide = 0.0;
#pragma unroll
                            for (int i = 0; i < kRopePairs; ++i) wide += static_cast<double>(x0[i]) * x0[i] + static_cast<double>(x1[i]) * x1[i];
#pragma unroll
                            for (int o = 16; o; o >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, o);
                            inv = static_cast<float>(1.0 / sqrt(wide / D + static_cast<double>(P.eps)));
                        }
#pragma unroll
                        for (int i = 0; i < kRopePairs; ++i) {
                            if (!l.is[i]) continue;
                            x0[i] = x0[i] * inv * P.q_norm[l.e0[i]];
                            x1[i] = x1[i] * inv * P.q_norm[l.e1[i]];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kRopePairs; ++i) {
                        if (!l.is[i]) continue;
                        y[l.e0[i]] = row_number<T>(l.turned[i] ? x0[i] * cs[i] - x1[i] * sn[i] : x0[i]);
                        y[l.e1[i]] = row_number<T>(l.turned[i] ? x1[i] * cs[i] + x0[i] * sn[i] : x1[i]);
                    }
                }
            }
        }
        __syncthreads();
    }
}

// ---- many tokens of a page: a lane has eight pairs of a head, so that rows are read and written by 16 bytes ---------------------------------
// The pairs 8 c .. 8 c + 7 of a head of D elements, c the lane's place in a group of G lanes (a power of two, some without pairs): their elements are eight at a
// and eight at b, pair by pair (apart: the rotation's halves) or one pair behind the other.
// (5,003 tokens of 128: 186 us by the kernel above, 74 by this one; by four pairs a lane a tenth to a half slower.)
struct RopeEight {
    int a, b, first;            // first: pair
    bool is, apart, turned;     // turned: all of them, or none
};
template <bool APART>
__device__ __forceinline__ RopeEight rope_eight(const KvRope &P, int c) {
    RopeEight e;
    const int half = P.rotary / 2;
    e.first = 8 * c;
    e.is = 16 * c < P.a.s.head_dim;
    e.turned = APART || e.first < half;
    e.apart = APART || (e.turned && !P.neighbours);
    e.a = e.apart ? e.first : 16 * c;
    e.b = e.apart ? half + e.first : 16 * c + 8;
    return e;
}
// eight numbers at a, eight at b, as they were read
template <class T>
struct RopeRaw {
    uint4 a[8 * sizeof(T) / 16], b[8 * sizeof(T) / 16];
    __device__ __forceinline__ void read(const T *row, const RopeEight &e, bool is) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) {
            a[i] = b[i] = make_uint4(0u, 0u, 0u, 0u);
            if (is) a[i] = reinterpret_cast<const uint4 *>(row + e.a)[i], b[i] = reinterpret_cast<const uint4 *>(row + e.b)[i];
        }
    }
    // the eight pairs' first and second elements
    __device__ __forceinline__ void pairs(const RopeEight &e, float *x0, float *x1) const {
        constexpr int N = 16 / sizeof(T);
        float at_a[8], at_b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            at_a[i] = static_cast<float>(reinterpret_cast<const T *>(&a[i / N])[i % N]);
            at_b[i] = static_cast<float>(reinterpret_cast<const T *>(&b[i / N])[i % N]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x0[i] = e.apart ? at_a[i] : i < 4 ? at_a[2 * i] : at_b[2 * i - 8];
            x1[i] = e.apart ? at_b[i] : i < 4 ? at_a[2 * i + 1] : at_b[2 * i - 7];
        }
    }
};
template <class T>
__device__ __forceinline__ void rope_put8(T *to, const float *x) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
        __align__(16) T y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = row_number<T>(x[i * N + j]);
        reinterpret_cast<uint4 *>(to)[i] = *reinterpret_cast<const uint4 *>(y);
    }
}
// eight pairs as they lie: at a, at b
__device__ __forceinline__ void rope_places(const RopeEight &e, const float *y0, const float *y1, float *a, float *b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] = e.apart ? y0[i] : i & 1 ? y1[i / 2] : y0[i / 2];
        b[i] = e.apart ? y1[i] : i & 1 ? y1[4 + i / 2] : y0[4 + i / 2];
    }
}

// sine and cosine of 2 pi turn, |turn| <= 1/2: those of the nearest 256th of a turn, from the table, and the series of the rest, put together; off by 2^-51
__device__ __forceinline__ void rope_sincos(const double2 *circle, double turn, double &sn, double &cs) {
    constexpr double magic = 6755399441055744.0;         // 1.5 2^52: what is added to it is rounded to a whole number
    const double t = 256.0 * turn, whole = t + magic, x = (t - (whole - magic)) * (6.283185307179586476925 / 256), x2 = x * x;
    const double2 at = circle[__double2loint(whole) & 255];
    const double s = fma(x2 * x, fma(x2, fma(x2, -1.0 / 5040, 1.0 / 120), -1.0 / 6), x), c = x2 * fma(x2, fma(x2, -1.0 / 720, 1.0 / 24), -0.5);         // (c: less 1)
    sn = at.y + fma(at.y, c, at.x * s);
    cs = at.x + fma(at.x, c, -(at.y * s));
}

constexpr int kRopeThreads = 256;
// (APART: all pairs are turned, and are of halves: known when it is compiled. 4,000 tokens of 32 x 64: 7 % faster)
template <class T, bool E4M3, bool APART>
__global__ void __launch_bounds__(kRopeThreads, 2) kv_rope_rows_kernel(const __grid_constant__ KvRope P) {
    extern __shared__ __align__(16) uint8_t rope_sm[];           // keys: rotated rows; values: the codes of the sub-blocks that the rows touch
    __shared__ double2 circle[256];                              // cosine and sine of a turn's 256ths
    __shared__ float part[kRopeThreads / 32];
    __shared__ int bad_any;
    const int n_seq = P.a.book[0], n_items = P.a.book[2], h = blockIdx.y, D = P.a.s.head_dim, tid = threadIdx.x;
    if (blockIdx.z == 0) {
        for (int i = tid; i < 256; i += kRopeThreads) sincospi(i / 128.0, &circle[i].y, &circle[i].x);
        __syncthreads();
    }
    const int shift = D <= 32 ? 1 : D <= 64 ? 2 : D <= 128 ? 3 : 4, G = 1 << shift, c = tid & (G - 1);
    const unsigned group = ((1u << G) - 1) << (tid & 31 & -G);          // the lanes of a head: a warp's groups may have tokens or not
    const RopeEight e = rope_eight<APART>(P, c);
    const float over_d = 1.0f / D;
    double turns[8];
    float w0[8], w1[8];
    const float *norm = blockIdx.z == 0 ? P.k_norm : P.q_norm;
    if (blockIdx.z != 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = e.first + i;
            turns[i] = e.is && e.turned ? P.turns[p] : 0.0;
            w0[i] = w1[i] = 1.0f;
            if (norm && e.is) w0[i] = norm[e.apart ? e.a + i : 2 * p], w1[i] = norm[e.apart ? e.b + i : 2 * p + 1];
        }
    }
    // less whole turns; first: the position on the first axis
    auto first_at = [&](int row, int place) { return static_cast<double>(P.positions ? P.positions[static_cast<size_t>(row) * P.n_axes] : place); };
    auto turn_of = [&](int i, double first, int row) {
        double at = first;
        if (P.n_axes > 1 && P.positions) {
            const int p = e.first + i, axis = min((p >= P.section_end[0]) + (p >= P.section_end[1]) + (p >= P.section_end[2]), P.n_axes - 1);
            at = static_cast<double>(P.positions[static_cast<size_t>(row) * P.n_axes + axis]);
        }
        const double a = at * turns[i];
        return a - rint(a);
    };
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const KvPagePart at = kv_page_part(P.a.book, P.a.table, P.a.s, n_seq, item);
        const int n = at.b - at.a;
        if (blockIdx.z == 1) {
            kv_append_part<T, E4M3, kRopeThreads>(P.a, at, h, 1, rope_sm, part, bad_any);
        } else if (blockIdx.z == 0) {
            const T *rows = static_cast<const T *>(P.a.rows[0]) + static_cast<size_t>(at.row) * P.a.stride[0] + static_cast<size_t>(h) * D;
            float *held = reinterpret_cast<float *>(rope_sm);
            auto rotate = [&](int t0, int m) {
                RopeRaw<T> raw;
                raw.read(rows + static_cast<size_t>(t0 + (tid >> shift)) * P.a.stride[0], e, e.is && tid >> shift < m);
#pragma unroll 1
                for (int t = tid >> shift; t < m; t += kRopeThreads >> shift) {
                    const int row = at.row + t0 + t, next = t + (kRopeThreads >> shift);
                    const double first = first_at(row, at.place + t0 + t);
                    float x0[8], x1[8];
                    raw.pairs(e, x0, x1);
                    raw.read(rows + static_cast<size_t>(t0 + next) * P.a.stride[0], e, e.is && next < m);
                    double inv = 1.0;
                    if (P.k_norm) {
                        double sum = 0.0, more = 0.0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum = fma(static_cast<double>(x0[i]), static_cast<double>(x0[i]), sum), more = fma(static_cast<double>(x1[i]), static_cast<double>(x1[i]), more);
                        sum += more;
                        for (int o = G / 2; o; o >>= 1) sum += __shfl_xor_sync(group, sum, o);
                        inv = rsqrt(sum / D + static_cast<double>(P.eps));
                    }
                    float a[8], b[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        double n0 = x0[i], n1 = x1[i];
                        if (P.k_norm) n0 = n0 * inv * w0[i], n1 = n1 * inv * w1[i];
                        if (e.turned) {
                            double sn, cs;
                            rope_sincos(circle, turn_of(i, first, row), sn, cs);
                            const double f = P.factor, y0 = f * (n0 * cs - n1 * sn), y1 = f * (n1 * cs + n0 * sn);
                            n0 = y0, n1 = y1;
                        }
                        x0[i] = static_cast<float>(n0);
                        x1[i] = static_cast<float>(n1);
                    }
                    rope_places(e, x0, x1, a, b);
                    if (e.is) {
#pragma unroll
                        for (int i = 0; i < 8; i += 4) {
                            *reinterpret_cast<float4 *>(held + rope_held(t * D + e.a + i)) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
                            *reinterpret_cast<float4 *>(held + rope_held(t * D + e.b + i)) = make_float4(b[i], b[i + 1], b[i + 2], b[i + 3]);
                        }
                    }
                }
            };
            auto load = [&](int t, int k, float *x) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 v = *reinterpret_cast<const float4 *>(held + rope_held(t * D + k + 4 * j));
                    x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
                }
            };
            float top = 0.0f;
            int bad = 0;
            for (int t0 = 0; t0 < n; t0 += P.held) {
                if (t0 > 0) __syncthreads();
                rotate(t0, min(P.held, n - t0));
                __syncthreads();
                top = kv_part_top<kRopeThreads>(D, min(P.held, n - t0), load, top, bad);
            }
            const KvPartScale sc = kv_part_scale<E4M3, kRopeThreads>(P.a, at, h, 0, top, bad, part, bad_any);
            for (int t0 = 0; t0 < n; t0 += P.held) {
                if (n > P.held) {
                    __syncthreads();
                    rotate(t0, min(P.held, n - t0));
                    __syncthreads();
                }
                kv_part_codes<E4M3, kRopeThreads>(P.a, at, h, 0, sc, nullptr, t0, min(P.held, n - t0), load);
            }
            kv_part_end(P.a, at, h, 0, sc.s, make_int2(0, 0));
        } else {
            const int g = P.a.s.heads / P.a.s.kv_heads, part_q = blockIdx.z - 2, h0 = h * g + g * part_q / P.q_parts, h1 = h * g + g * (part_q + 1) / P.q_parts;
            // where there are fewer tokens than groups, some groups share one's heads
            const int groups = kRopeThreads >> shift, share = n < groups ? min(h1 - h0, groups / n) : 1, slot = tid >> shift;
            constexpr int B = 4 / sizeof(T);        // heads that are asked for at once: of 32 bits one, of 16 bits two (5,003 tokens of 32 x 128: 75 us for 84 one by one)
#pragma unroll 1
            for (int t = slot / share; t < n; t += groups / share) {
                const T *from = static_cast<const T *>(P.q) + static_cast<size_t>(at.row + t) * P.q_stride;
                T *to = static_cast<T *>(P.q_out) + static_cast<size_t>(at.row + t) * P.q_out_stride;
                RopeRaw<T> raw[B];
                auto ask = [&](int head) {
#pragma unroll
                    for (int j = 0; j < B; ++j) raw[j].read(from + static_cast<size_t>(head + j * share) * D, e, e.is && head + j * share < h1);
                };
                ask(h0 + slot % share);
                const double first = first_at(at.row + t, at.place + t);
                float cs[8], sn[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    cs[i] = 1.0f, sn[i] = 0.0f;
                    if (e.turned) {
                        sincospif(static_cast<float>(2.0 * turn_of(i, first, at.row + t)), &sn[i], &cs[i]);
                        cs[i] *= P.factor, sn[i] *= P.factor;
                    }
                }
                auto one = [&](const RopeRaw<T> &raw, int head) {
                    float x0[8], x1[8];
                    raw.pairs(e, x0, x1);
                    if (P.q_norm) {
                        float sum = 0.0f, more = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) sum = fmaf(x0[i], x0[i], sum), more = fmaf(x1[i], x1[i], more);
                        sum += more;
                        for (int o = G / 2; o; o >>= 1) sum += __shfl_xor_sync(group, sum, o);
                        float inv = rsqrtf(fmaf(sum, over_d, P.eps));
                        if (!(sum > 1e-30f && sum < 1e38f)) {           // squares that F32 does not hold
                            double wide = 0.0;
#pragma unroll
                            for (int i = 0; i < 8; ++i) wide += static_cast<double>(x0[i]) * x0[i] + static_cast<double>(x1[i]) * x1[i];
                            for (int o = G / 2; o; o >>= 1) wide += __shfl_xor_sync(group, wide, o);
                            inv = static_cast<float>(1.0 / sqrt(wide / D + static_cast<double>(P.eps)));
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) x0[i] = x0[i] * inv * w0[i], x1[i] = x1[i] * inv * w1[i];
                    }
                    float y0[8], y1[8], a[8], b[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        y0[i] = e.turned ? x0[i] * cs[i] - x1[i] * sn[i] : x0[i];
                        y1[i] = e.turned ? x1[i] * cs[i] + x0[i] * sn[i] : x1[i];
                    }
                    rope_places(e, y0, y1, a, b);
                    if (e.is) {
                        rope_put8(to + static_cast<size_t>(head) * D + e.a, a);
                        rope_put8(to + static_cast<size_t>(head) * D + e.b, b);
                    }
                };
#pragma unroll 1
                for (int head = h0 + slot % share; head < h1;) {
#pragma unroll
                    for (int j = 0; j < B; ++j)
                        if (head + j * share < h1) one(raw[j], head + j * share);
                    head += B * share;
                    if (head < h1) ask(head);
                }
            }
        }
        __syncthreads();
    }
}

}  // namespace
}  // namespace wd

extern "C" {

int wd_rope_create(const wd_rope_config *cfg, const double *inv_freq, wd_rope **out) {
    return wd_host::guarded([&]() -> int {
        if (!cfg || !out) return set_error(WD_E_INVALID, "null argument");
        *out = nullptr;
        wd_rope_config c = *cfg;
        if (c.rotary_dim == 0) c.rotary_dim = c.head_dim;
        if (c.n_axes == 0) c.n_axes = 1;
        if (c.head_dim < 2 || c.head_dim > 256) return set_error(WD_E_INVALID, "rotary positions: head_dim must be 2 to 256");
        if (c.rotary_dim < 2 || c.rotary_dim > c.head_dim || c.rotary_dim % 2) return set_error(WD_E_INVALID, "rotary positions: rotary_dim must be even, 2 to head_dim");
        if (c.pairs != WD_ROPE_HALVES && c.pairs != WD_ROPE_NEIGHBOURS) return set_error(WD_E_INVALID, "rotary positions: pairs must be WD_ROPE_HALVES or WD_ROPE_NEIGHBOURS");
        if (c.n_axes < 1 || c.n_axes > 4) return set_error(WD_E_INVALID, "rotary positions: 1 to 4 axes");
        if (!std::isfinite(c.factor) || !(inv_freq || (c.theta > 0.0f && std::isfinite(c.theta)))) return set_error(WD_E_INVALID, "rotary positions: theta must be positive, factor finite");
        auto r = std::make_unique<wd_rope>();
        const int pairs = c.rotary_dim / 2;
        int end = 0;
        for (int i = 0; i < 4; ++i) {
            if (c.n_axes > 1 && i < c.n_axes) {
                if (c.sections[i] < 0 || c.sections[i] > pairs - end) return set_error(WD_E_INVALID, "rotary positions: the axes' pairs must be rotary_dim / 2 together");
                end += c.sections[i];
            } else {
                end = i < c.n_axes ? pairs : end;
            }
            r->section_end[i] = end;
        }
        if (end != pairs) return set_error(WD_E_INVALID, "rotary positions: the axes' pairs must be rotary_dim / 2 together");
        for (int p = 0; p < pairs; ++p) {
            const double f = inv_freq ? inv_freq[p] : std::pow(static_cast<double>(c.theta), -2.0 * p / c.rotary_dim);
            if (!std::isfinite(f)) return set_error(WD_E_INVALID, "rotary positions: frequencies must be finite");
            r->turns[p] = f / 6.283185307179586476925;
        }
        r->cfg = c;
        *out = r.release();
        return WD_OK;
    });
}

void wd_rope_destroy(wd_rope *r) { delete r; }

int wd_kv_append_rope(wd_kv_cache *c, int layer, const wd_rope *r, const wd_rope_rows *x, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (int rc = check_device(c)) return rc;
        if (!r || !x) return set_error(WD_E_INVALID, "null argument");
        if (layer < 0 || layer >= c->cfg.n_layers) return set_error(WD_E_INVALID, "key/value cache: layer out of range");
        if (r->cfg.head_dim != c->cfg.head_dim) return set_error(WD_E_INVALID, "key/value cache: rotary positions of another head_dim");
        if ((x->q_norm_dev || x->k_norm_dev) && !(x->eps > 0.0f && std::isfinite(x->eps))) return set_error(WD_E_INVALID, "key/value cache: eps of the norms must be positive");
        if ((x->q_dev == nullptr) != (x->q_out_dev == nullptr)) return set_error(WD_E_INVALID, "key/value cache: q needs its output, and the other way round");
        for (const void *p : {static_cast<const void *>(x->positions_dev), static_cast<const void *>(x->q_norm_dev), static_cast<const void *>(x->k_norm_dev)})
            if (reinterpret_cast<uintptr_t>(p) % 4) return set_error(WD_E_INVALID, "key/value cache: positions and norms are not aligned to their type");
        int rows_of = 0;
        if (int rc = rows_type(x->type, &rows_of)) return rc;
        if (c->book[0] == 0) return set_error(WD_E_STATE, "key/value cache: no step has begun");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c->items == 0) return check_not_captured(c, s);
        const size_t size = rows_size(rows_of);
        const int D = c->cfg.head_dim, H = c->cfg.n_kv_heads, g = c->cfg.n_heads / H;
        const long long width = static_cast<long long>(H) * D;
        wd::KvRope p;
        p.a.stride[0] = x->k_stride;
        p.a.stride[1] = x->v_stride;
        if (int rc = check_rows(x->k_dev, size, &p.a.stride[0], width, "k")) return rc;
        if (int rc = check_rows(x->v_dev, size, &p.a.stride[1], width, "v")) return rc;
        p.q_stride = x->q_stride;
        p.q_out_stride = x->q_out_stride;
        if (x->q_dev) {
            if (int rc = check_rows(x->q_dev, size, &p.q_stride, width * g, "q")) return rc;
            if (int rc = check_rows(x->q_out_dev, size, &p.q_out_stride, width * g, "q's output")) return rc;
            if (x->q_dev == x->q_out_dev && p.q_stride != p.q_out_stride) return set_error(WD_E_INVALID, "key/value cache: an output over q needs q's stride");
        }
        OnDevice on(c->cfg.device);
        if (int rc = note_capture(c, s)) return rc;
        fill_append(c, layer, x->k_dev, x->v_dev, size, &p.a);
        p.q = x->q_dev;
        p.q_out = x->q_out_dev;
        p.positions = x->positions_dev;
        p.q_norm = x->q_norm_dev;
        p.k_norm = x->k_norm_dev;
        p.eps = x->eps;
        p.factor = r->cfg.factor;
        p.rotary = r->cfg.rotary_dim;
        p.neighbours = r->cfg.pairs == WD_ROPE_NEIGHBOURS;
        p.n_axes = r->cfg.n_axes;
        for (int i = 0; i < 4; ++i) p.section_end[i] = r->section_end[i];
        for (int i = 0; i < 128; ++i) p.turns[i] = r->turns[i];
        const int most = std::min(c->max_rows, c->cfg.page_tokens);       // of a page (a replay may have more)
        p.held = std::min(most, wd::kRopeHeld / D);
        const size_t smem = std::max<size_t>(static_cast<size_t>(p.held) * D * 4, static_cast<size_t>(c->cfg.page_tokens) * D);
        // one head of q a block where there are not enough blocks for the SMs, all that share a kv head where there are
        p.q_parts = std::max<long long>(1, std::min<long long>(g, 4ll * c->n_sm / (static_cast<long long>(c->items) * H)));
        const dim3 grid(static_cast<unsigned>(c->items), H, x->q_dev ? 2 + p.q_parts : 2);
        const bool small = static_cast<long long>(most) * D <= 2048;
        // by eights of pairs where the rows lie on boundaries of 16 bytes and no eight has some pairs that are turned and some that are not
        bool by_eight = !small && r->cfg.rotary_dim % 16 == 0 && p.a.vec[0];
        if (x->q_dev) by_eight &= (reinterpret_cast<uintptr_t>(x->q_dev) | reinterpret_cast<uintptr_t>(x->q_out_dev)) % 16 == 0 && p.q_stride * size % 16 == 0 && p.q_out_stride * size % 16 == 0;
        return by_rows_and_codes(c, rows_of, [&](auto t, auto e4m3) {
            using T = decltype(t);
            auto launch = [&](auto kernel, int threads) {
                // (the attribute is the kernel's, for all threads and caches: never what this call needs alone)
                WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, wd::kRopeHeld * 4));
                kernel<<<grid, threads, smem, s>>>(p);
                WD_TRY_CUDA(cudaGetLastError());
                return WD_OK;
            };
            if (by_eight && !p.neighbours && p.rotary == D) return launch(wd::kv_rope_rows_kernel<T, decltype(e4m3)::value, true>, wd::kRopeThreads);
            if (by_eight) return launch(wd::kv_rope_rows_kernel<T, decltype(e4m3)::value, false>, wd::kRopeThreads);
            return small ? launch(wd::kv_rope_kernel<T, decltype(e4m3)::value, 64>, 64) : launch(wd::kv_rope_kernel<T, decltype(e4m3)::value, 256>, 256);
        });
    });
}

}  // extern "C"
