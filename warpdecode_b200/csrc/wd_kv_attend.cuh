// Attention over the 8-bit cache for few rows: the last tokens of each of a step's sequences against everything in front of them.
//
//   out[r] = sum_j p_j cv_j sv_j / sum_j p_j,   p_j = 2^(x_j - m),   x_j = (q[r] . ck_j) (2^e scale log2(e) sk_j)
//
// q is brought to F16 row by row: q = 2^e (hi + lo) with |hi| <= 1, lo = 0 unless the rows are F32; codes are exact in F16; sums are F32.
// The scales of the values go into the exponent: m is the running maximum of x_j + log2(sv_j), P_j = 2^(x_j + log2 sv_j - m) <= 1 is what meets the
// codes (F16, hi + lo for F32 rows), and the denominator takes P_j / sv_j in F32. A page whose values are small loses nothing beside one whose values
// are large unless its part of the sum is small.
//
// Products: keys and values are the A operands (16 tokens, or 16 elements of the head), 8 rows of q the B operand, so that a group of up to 8 query
// heads wastes nothing and the codes are expanded once for all of a warp's rows. The weights come out of the first product with tokens along the
// lanes' g and are needed with tokens along t: one 8 x 8 transposition of F16 pairs (movmatrix) each.
//
// Work: a tile is 64 tokens of one kv head, an item the tiles that 8 N8 rows of a head of a sequence see. All items' tiles are numbered through
// (an item counts a few more than it has, for what it costs to begin and end one), and each worker, a warp, takes an equal run of the numbers, whatever
// the sequences' lengths. A worker has a warp beside it that brings its keys and values into a ring of its own by bulk copies. Nothing is waited for
// between workers until all of a CTA's are done; then the parts of items that several of them hold are put together, and those that several CTAs
// hold by the last CTA to arrive, always in the workers' order.
#pragma once

#include "wd_kv_layout.cuh"

namespace wd {

constexpr int kAttWorkers = 8, kAttThreads = 512, kAttMaxSeqs = 1024, kAttMaxRows = 16, kAttMaxSlots = 8;
// Registers a thread: the warps that compute take what those that copy give back (128 at launch).
constexpr int kAttRegsMore = 192, kAttRegsLess = 64;
static_assert(256 * kAttRegsMore + 256 * kAttRegsLess <= kAttThreads * 128, "more than the block was launched with: the increase would wait for ever");
constexpr float kAttFloor = -1.0e30f;       // a maximum over nothing

struct KvAttend {
    const uint8_t *pool;        // of the layer
    const float *scales;        // of the layer
    const int *book;
    const int *table;
    const void *q;
    void *out;
    long long q_stride, out_stride;
    float *part;                // [workers][2][kAttMaxRows][D + 4]: sums, then maximum and denominator
    float *cta_part;            // [CTAs][2][kAttMaxRows][D + 4]
    unsigned *arrived;          // [CTAs]
    unsigned *status;
    float scale_log2;
    int type, window, workers, slots;
    KvShape s;
};

template <int D>
struct AttendPlan {
    static constexpr int kCw = D % 64 == 0 ? 64 : 32;
    static constexpr int kSlot = 64 * D + 64;           // keys or values of a tile; behind the keys 4 x {key scale, log2 of the value scale, 1 / value scale}
    __host__ __device__ static constexpr int q_bytes(int n8, bool split) { return n8 * 8 * D * 2 * (split ? 2 : 1); }
    __host__ __device__ static constexpr int fixed_bytes(int workers, int n8, bool split) { return workers * q_bytes(n8, split) + (kAttMaxSeqs + 2) * 8; }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void att_bar() { asm volatile("bar.sync 1, %0;" ::"n"(kAttWorkers * 32) : "memory"); }
// two floats -> F16 pair, and the pair of what that rounding left over
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t half_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return half_pair(a - f.x, b - f.y);
}

// Bounded wait by a count of polls, inline (a call would keep the compiler from moving registers between the warpgroups): a poll suspends the thread
// for 1.3 us, so that the limit is 1.4 s, or 0.3 ms once another wait has run out. What follows reads what is there and ends.
__device__ __forceinline__ void att_wait(uint64_t *bar, uint32_t parity, unsigned *status) {
#pragma unroll 1
    for (unsigned i = 0; i < kSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 255u) == 255u && *reinterpret_cast<volatile unsigned *>(status) & kErrCopyTimeout) break;
    }
    atomicOr(status, kErrCopyTimeout);
}

// A run's part of an item.
struct AttSegment {
    int seq, row0, count, length, head, item_row, rows;         // rows: of the item, from item_row on
    int lo, hi;                 // tiles of 64 tokens, absolute
    int whole;                  // the run holds all of the item
    long long item0, item1, next;       // numbers: the item's, and the one behind the segment
};

// Tiles that an item of a sequence counts: the most that any of its row groups can see.
__device__ __forceinline__ int att_tiles(int length, int count, int group_rows, int g, int window) {
    const int all = (length + 63) >> 6;
    if (window == 0) return all;
    const int tokens = min(count, (group_rows + g - 1) / g + 1);
    return min(all, (min(window, length) + tokens + 62) / 64 + 1);
}

template <int D, int N8, bool SPLIT, bool E4M3>
__global__ void __launch_bounds__(kAttThreads, 1) kv_attend_kernel(const __grid_constant__ KvAttend P) {
    using A = AttendPlan<D>;
    constexpr int CW = A::kCw, LB = CW / 4, NH = LB / 8, ROWS = 8 * N8, PITCH = D + 4;
    extern __shared__ __align__(128) uint8_t att_sm[];
    __shared__ __align__(8) uint64_t full[kAttWorkers][kAttMaxSlots], empty[kAttWorkers][kAttMaxSlots];
    __shared__ long long part_item[kAttWorkers * 2][2];          // first and last number of the item that a worker's first or last part belongs to; -1: none
    __shared__ int4 part_rows[kAttWorkers * 2];                 // row0, head, item_row, rows
    __shared__ int run_first[kAttWorkers * 2], run_last[kAttWorkers * 2], n_runs, last_one[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), worker = warp & 7;
    uint8_t *ring = att_sm + worker * P.slots * A::kSlot;
    uint8_t *qs = att_sm + P.workers * (P.slots * A::kSlot + 0) + worker * A::q_bytes(N8, SPLIT);
    long long *prefix = reinterpret_cast<long long *>(att_sm + P.workers * (P.slots * A::kSlot + A::q_bytes(N8, SPLIT)));
    const int n_seq = P.book[0], g_heads = P.s.heads / P.s.kv_heads;
    const int *entries = P.book + kKvHead;
    if (tid < kAttWorkers * kAttMaxSlots) {
        mbar_init(&full[tid / kAttMaxSlots][tid % kAttMaxSlots], 1);
        mbar_init(&empty[tid / kAttMaxSlots][tid % kAttMaxSlots], 1);
        mbar_fence_init();
    }
    if (tid < kAttWorkers * 2) part_item[tid][0] = -1;
    // numbers of one head in front of each sequence, without what an item costs beside its tiles: items in the upper half of a word
    if (warp == 0) {
        long long sum = 0;
        for (int i0 = 0; i0 < n_seq; i0 += 32) {
            const int i = i0 + lane;
            long long v = 0;
            if (i < n_seq) {
                const int *e = entries + i * kKvStepWords;
                const long long items = (static_cast<long long>(e[2]) * g_heads + ROWS - 1) / ROWS;
                v = items * att_tiles(e[3], e[2], ROWS, g_heads, P.window);
            }
            long long inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            if (i < n_seq) prefix[i] = sum + inc - v;
            sum += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) prefix[n_seq] = sum;
    }
    __syncthreads();
    const int all_workers = static_cast<int>(gridDim.x) * P.workers, me = static_cast<int>(blockIdx.x) * P.workers + worker;
    // what an item costs beside its tiles, in tiles: next to nothing where each worker has one part of one item anyway
    const long long tiles = prefix[n_seq] * P.s.kv_heads;
    const int extra = tiles >= 2ll * all_workers ? 2 : 0;
    if (extra > 0) {
        __syncthreads();
        if (warp == 0) {
            long long sum = 0;
            for (int i0 = 0; i0 < n_seq; i0 += 32) {
                const int i = i0 + lane;
                long long v = i < n_seq ? (static_cast<long long>(entries[i * kKvStepWords + 2]) * g_heads + ROWS - 1) / ROWS * extra : 0, inc = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += y;
                }
                if (i < n_seq) prefix[i] += sum + inc - v;
                sum += __shfl_sync(0xffffffffu, inc, 31);
            }
            if (lane == 0) prefix[n_seq] += sum;
        }
        __syncthreads();
    }
    const long long total = prefix[n_seq] * P.s.kv_heads;
    if (total == 0) return;
    const long long chunk = (total + all_workers - 1) / all_workers, cta_chunk = chunk * P.workers;
    if (blockIdx.x * cta_chunk >= total) return;
    const long long begin = worker < P.workers ? min(me * chunk, total) : total, end = min(begin + chunk, total);

    auto segment = [&](long long at) {
        AttSegment s;
        int lo = 0, hi = n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] * P.s.kv_heads <= at) lo = mid;
            else hi = mid - 1;
        }
        const int *e = entries + lo * kKvStepWords;
        s.seq = e[0], s.row0 = e[1], s.count = e[2], s.length = e[3];
        const int per_item = att_tiles(s.length, s.count, ROWS, g_heads, P.window) + extra;
        const long long per_head = prefix[lo + 1] - prefix[lo], base = prefix[lo] * P.s.kv_heads, in = at - base;
        s.head = static_cast<int>(in / per_head);
        const int group = static_cast<int>((in - s.head * per_head) / per_item);
        s.item0 = base + s.head * per_head + static_cast<long long>(group) * per_item;
        s.item1 = s.item0 + per_item;
        s.item_row = group * ROWS;
        s.rows = min(ROWS, s.count * g_heads - s.item_row);
        s.next = min(s.item1, end);
        s.whole = s.item0 >= begin && s.item1 <= end;
        const int pos0 = s.length - s.count + s.item_row / g_heads, pos1 = s.length - s.count + (s.item_row + s.rows - 1) / g_heads;
        const int low = P.window ? max(0, pos0 - P.window + 1) >> 6 : 0, high = (pos1 >> 6) + 1;
        s.lo = min(low + max(0, static_cast<int>(at - s.item0) - extra), high);
        s.hi = min(low + max(0, static_cast<int>(s.next - s.item0) - extra), high);
        return s;
    };

    if (warp >= kAttWorkers) {
        // ---- copies: lane 4 j + i looks up sub-block i of the j-th of eight tiles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAttRegsLess));
        int slot = 0;
        uint32_t par = 1;
        const int shift = P.s.page_shift, grain = min(shift, 6), subs = 1 << (grain - 4);      // a copy is a page's tokens, 64 at most
        const uint32_t bytes = static_cast<uint32_t>(D) << grain;
        uint64_t *fu = full[worker], *em = empty[worker];
#pragma unroll 1
        for (long long at = begin; at < end;) {
            const AttSegment s = segment(at);
            at = s.next;
            const int *table = P.table + static_cast<size_t>(s.seq) * P.s.max_pages;
            const int last_sub = (s.length - 1) >> 4;
            const uint8_t *src = nullptr;
            float2 sc = make_float2(0.0f, 0.0f);
            auto look_up = [&](int tile0) {
                const int sub = min(4 * tile0 + lane, last_sub);            // behind the last one: the last one again, whose tokens are not seen twice
                const int page = table[sub >> (shift - 4)];
                src = P.pool + static_cast<size_t>(page) * kv_page_bytes(P.s) + s.head * kv_head_bytes(P.s) +
                      (sub & ((1 << (shift - 4)) - 1) & ~(subs - 1)) * kv_sub_bytes(D);
                sc = *reinterpret_cast<const float2 *>(P.scales + (static_cast<size_t>(page) * P.s.kv_heads + s.head) * 2);
            };
            if (s.lo < s.hi) look_up(s.lo);
#pragma unroll 1
            for (int t0 = s.lo; t0 < s.hi; t0 += 8) {
                const uint8_t *now = src;
                const float v = sc.y > 0.0f ? sc.y : kKvLeastScale;         // 0: nothing but zeros
                const float4 mine = make_float4(sc.x, log2f(v), 1.0f / v, 0.0f);
                if (t0 + 8 < s.hi) look_up(t0 + 8);
#pragma unroll 1
                for (int j = 0; j < 8 && t0 + j < s.hi; ++j) {
                    const bool copies = (lane >> 2) == j && (lane & (subs - 1)) == 0;
                    const int i = lane & 3;
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv) {
                        att_wait(&em[slot], par, P.status);
                        uint8_t *dst = ring + slot * A::kSlot;
                        if (kv == 0 && (lane >> 2) == j) *reinterpret_cast<float4 *>(dst + 64 * D + i * 16) = mine;
                        __syncwarp();
                        if (lane == 4 * j) mbar_expect_tx(&fu[slot], 64 * D);
                        __syncwarp();
                        if (copies) bulk_load(dst + i * 16 * D, now + kv * kv_half_bytes(P.s), bytes, &fu[slot]);
                        if (++slot == P.slots) {
                            slot = 0;
                            par ^= 1;
                        }
                    }
                }
            }
        }
        return;
    }

    // ---- the warps that compute
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAttRegsMore));
    const int g = lane >> 2, t = lane & 3;
    int slot = 0;
    uint32_t par = 0;
    uint64_t *fu = full[worker], *em = empty[worker];
    auto pass_on = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&em[slot]);
        if (++slot == P.slots) {
            slot = 0;
            par ^= 1;
        }
    };
#pragma unroll 1
    for (long long at = begin; at < end;) {
        const AttSegment s = segment(at);
        const bool first_part = at == begin;
        at = s.next;
        // q -> fragments: [8 rows][D / CW][half of LB][lane][8 elements], hi, then lo
        float mul[N8][2];
        __syncwarp();
#pragma unroll
        for (int n = 0; n < N8; ++n) {
#pragma unroll
            for (int rb = 0; rb < 8; rb += 4) {
                float x[4][D / 32];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 8 * n + rb + j, row = s.item_row + r;
                    const size_t src = static_cast<size_t>(s.row0 + row / g_heads) * P.q_stride + (static_cast<size_t>(s.head) * g_heads + row % g_heads) * D;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) x[j][i] = r < s.rows ? row_load(P.q, P.type, src + i * 32 + lane) : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int gr = rb + j;
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) top = fmaxf(top, fabsf(x[j][i]));
#pragma unroll
                    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const int e = top > 0.0f ? max(-100, min(128, static_cast<int>(__float_as_uint(top) >> 23) - 126)) : 0, e1 = e / 2, e2 = e - e1;
                    const float up = __uint_as_float((127 + e1) << 23), up2 = __uint_as_float((127 + e2) << 23), down = __uint_as_float((127 - e1) << 23),
                                down2 = __uint_as_float((127 - e2) << 23);
                    if ((gr >> 1) == t) mul[n][gr & 1] = P.scale_log2 * up * up2;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const int d = i * 32 + lane, kk = d % CW, el = kk % LB;
                        const float v = x[j][i] * down * down2;
                        const __half hi = __float2half_rn(v);
                        __half *to = reinterpret_cast<__half *>(qs) + (((n * (D / CW) + d / CW) * NH + el / 8) * 32 + gr * 4 + kk / LB) * 8 + el % 8;
                        *to = hi;
                        if (SPLIT) to[ROWS * D] = __float2half_rn(v - __half2float(hi));
                    }
                }
            }
        }
        __syncwarp();
        float o[N8][D / 16][4], m[N8][2], l[N8][2];
        int pos[N8][2];
        const int start = s.length - s.count, last_row = s.item_row + s.rows - 1, pos_lo = start + s.item_row / g_heads, pos_hi = start + last_row / g_heads;
#pragma unroll
        for (int n = 0; n < N8; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[n][i] = kAttFloor;
                l[n][i] = 0.0f;
                pos[n][i] = start + min(s.item_row + 8 * n + 2 * t + i, last_row) / g_heads;
            }
        }
#pragma unroll 1
        for (int tile = s.lo; tile < s.hi; ++tile) {
            // tokens x rows: x[n][b][c] is token 16 b + g + 8 (c >> 1) of the tile, row 8 n + 2 t + (c & 1)
            float x[N8][4][4];
#pragma unroll
            for (int n = 0; n < N8; ++n)
#pragma unroll
                for (int b = 0; b < 4; ++b) x[n][b][0] = x[n][b][1] = x[n][b][2] = x[n][b][3] = 0.0f;
            att_wait(&fu[slot], par, P.status);
            const uint8_t *kp = ring + slot * A::kSlot + g * CW + t * LB;
            const uint4 *qp = reinterpret_cast<const uint4 *>(qs) + lane;
#pragma unroll
            for (int c = 0; c < D / CW; ++c) {
                uint4 qh[N8][NH], ql[SPLIT ? N8 : 1][NH];
#pragma unroll
                for (int n = 0; n < N8; ++n)
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        qh[n][h] = qp[((n * (D / CW) + c) * NH + h) * 32];
                        if constexpr (SPLIT) ql[n][h] = qp[((n * (D / CW) + c) * NH + h) * 32 + ROWS * D / 8];
                    }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t w0[LB / 4], w1[LB / 4];
                    const uint8_t *p = kp + b * 16 * D + c * 16 * CW;
                    if constexpr (LB == 16) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(p), v = *reinterpret_cast<const uint4 *>(p + 8 * CW);
                        w0[0] = u.x, w0[1] = u.y, w0[2] = u.z, w0[3] = u.w;
                        w1[0] = v.x, w1[1] = v.y, w1[2] = v.z, w1[3] = v.w;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2 *>(p), v = *reinterpret_cast<const uint2 *>(p + 8 * CW);
                        w0[0] = u.x, w0[1] = u.y;
                        w1[0] = v.x, w1[1] = v.y;
                    }
#pragma unroll
                    for (int w = 0; w < LB / 4; ++w) {
                        uint32_t a0, a1, a2, a3;
                        kv_halves<E4M3>(w0[w], a0, a2);
                        kv_halves<E4M3>(w1[w], a1, a3);
#pragma unroll
                        for (int n = 0; n < N8; ++n) {
                            const uint4 q = qh[n][w >> 1];
                            mma_f16(x[n][b], a0, a1, a2, a3, w & 1 ? q.z : q.x, w & 1 ? q.w : q.y);
                            if constexpr (SPLIT) {
                                const uint4 r = ql[n][w >> 1];
                                mma_f16(x[n][b], a0, a1, a2, a3, w & 1 ? r.z : r.x, w & 1 ? r.w : r.y);
                            }
                        }
                    }
                }
            }
            float4 sc[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) sc[b] = *reinterpret_cast<const float4 *>(ring + slot * A::kSlot + 64 * D + b * 16);
            pass_on();
            const int first = tile * 64;
            if (first + 63 > pos_lo || (P.window && first <= pos_hi - P.window)) {
#pragma unroll
                for (int n = 0; n < N8; ++n)
#pragma unroll
                    for (int b = 0; b < 4; ++b)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int token = first + 16 * b + g + 8 * (c >> 1), at_row = pos[n][c & 1];
                            if (token > at_row || (P.window && token <= at_row - P.window)) x[n][b][c] = -INFINITY;
                        }
            }
            uint32_t ph[N8][4][2], pl[SPLIT ? N8 : 1][4][2];
            bool grown = false;
            float f[N8][2];
#pragma unroll
            for (int n = 0; n < N8; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = kAttFloor;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        // (a scale of 0 makes every product 0; what is masked must not become 0 times -inf)
                        const float c = fmaxf(mul[n][i] * sc[b].x, 1e-37f);
                        top = fmaxf(top, fmaf(fmaxf(x[n][b][i], x[n][b][2 + i]), c, sc[b].y));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float now = fmaxf(m[n][i], top);
                    f[n][i] = ex2(m[n][i] - now);
                    grown |= now != m[n][i];
                    m[n][i] = now;
                    float sum = 0.0f;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const float c = fmaxf(mul[n][i] * sc[b].x, 1e-37f), off = sc[b].y - now;
                        x[n][b][i] = ex2(fmaf(x[n][b][i], c, off));
                        x[n][b][2 + i] = ex2(fmaf(x[n][b][2 + i], c, off));
                        sum = fmaf(x[n][b][i] + x[n][b][2 + i], sc[b].z, sum);
                    }
                    l[n][i] = fmaf(l[n][i], f[n][i], sum);
                }
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t hi = half_pair(x[n][b][2 * h], x[n][b][2 * h + 1]);
                        ph[n][b][h] = transposed(hi);
                        if constexpr (SPLIT) pl[n][b][h] = transposed(half_rest(x[n][b][2 * h], x[n][b][2 * h + 1], hi));
                    }
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int n = 0; n < N8; ++n)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) o[n][i][0] *= f[n][0], o[n][i][1] *= f[n][1], o[n][i][2] *= f[n][0], o[n][i][3] *= f[n][1];
            }
            att_wait(&fu[slot], par, P.status);
            const uint4 *vp = reinterpret_cast<const uint4 *>(ring + slot * A::kSlot) + lane;
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const uint4 v = vp[b * D + k * 32];
                    uint32_t a0, a1, a2, a3;
                    kv_halves<E4M3>(v.x, a0, a2);
                    kv_halves<E4M3>(v.y, a1, a3);
#pragma unroll
                    for (int n = 0; n < N8; ++n) {
                        mma_f16(o[n][2 * k], a0, a1, a2, a3, ph[n][b][0], ph[n][b][1]);
                        if constexpr (SPLIT) mma_f16(o[n][2 * k], a0, a1, a2, a3, pl[n][b][0], pl[n][b][1]);
                    }
                    kv_halves<E4M3>(v.z, a0, a2);
                    kv_halves<E4M3>(v.w, a1, a3);
#pragma unroll
                    for (int n = 0; n < N8; ++n) {
                        mma_f16(o[n][2 * k + 1], a0, a1, a2, a3, ph[n][b][0], ph[n][b][1]);
                        if constexpr (SPLIT) mma_f16(o[n][2 * k + 1], a0, a1, a2, a3, pl[n][b][0], pl[n][b][1]);
                    }
                }
            pass_on();
        }
        // ---- the item's end, or this worker's part of it
        const int place = worker * 2 + (first_part ? 0 : 1);
        float *part = P.part + (static_cast<size_t>(me) * 2 + (first_part ? 0 : 1)) * kAttMaxRows * PITCH;
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float den = l[n][i];
                den += __shfl_xor_sync(0xffffffffu, den, 4);
                den += __shfl_xor_sync(0xffffffffu, den, 8);
                den += __shfl_xor_sync(0xffffffffu, den, 16);
                const int r = 8 * n + 2 * t + i, row = s.item_row + r;
                if (r >= s.rows) continue;
                if (s.whole) {
                    const float inv = 1.0f / den;
                    const size_t to = static_cast<size_t>(s.row0 + row / g_heads) * P.out_stride + (static_cast<size_t>(s.head) * g_heads + row % g_heads) * D + g;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        row_store(P.out, P.type, to + 16 * k, o[n][k][i] * inv);
                        row_store(P.out, P.type, to + 16 * k + 8, o[n][k][2 + i] * inv);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        __stcg(part + r * PITCH + 16 * k + g, o[n][k][i]);
                        __stcg(part + r * PITCH + 16 * k + 8 + g, o[n][k][2 + i]);
                    }
                    if (g == 0) __stcg(reinterpret_cast<float2 *>(part + r * PITCH + D), make_float2(m[n][i], den));
                }
            }
        if (!s.whole && lane == 0) {
            part_item[place][0] = s.item0;
            part_item[place][1] = s.item1;
            part_rows[place] = make_int4(s.row0, s.head, s.item_row, s.rows);
        }
    }

    // ---- parts of the CTA's workers: runs of places that belong to one item
    __threadfence_block();
    att_bar();
    if (tid == 0) {
        int runs = 0;
        for (int p = 0; p < kAttWorkers * 2; ++p) {
            if (part_item[p][0] < 0) continue;
            if (runs > 0 && part_item[run_last[runs - 1]][0] == part_item[p][0]) {
                run_last[runs - 1] = p;
            } else {
                run_first[runs] = run_last[runs] = p;
                ++runs;
            }
        }
        n_runs = runs;
        last_one[0] = last_one[1] = -1;
    }
    att_bar();
    const int runs = n_runs;
    if (runs == 0) return;
    const long long cta0 = blockIdx.x * cta_chunk, cta1 = min(cta0 + cta_chunk, total);
    constexpr int V = D / 4;
    auto put = [&](const int4 &rw, int r, int c, const float4 &sum, float den) {
        const int row = rw.z + r;
        const size_t to = static_cast<size_t>(rw.x + row / g_heads) * P.out_stride + (static_cast<size_t>(rw.y) * g_heads + row % g_heads) * D + c;
        const float inv = 1.0f / den;
        row_store(P.out, P.type, to, sum.x * inv);
        row_store(P.out, P.type, to + 1, sum.y * inv);
        row_store(P.out, P.type, to + 2, sum.z * inv);
        row_store(P.out, P.type, to + 3, sum.w * inv);
    };
    auto join = [&](float &top, float &den, float4 &sum, const float *p, int c) {
        const float4 y = __ldcg(reinterpret_cast<const float4 *>(p + c));
        const float2 z = __ldcg(reinterpret_cast<const float2 *>(p + D));
        const float both = fmaxf(top, z.x), fa = ex2(top - both), fb = ex2(z.x - both);
        top = both;
        den = den * fa + z.y * fb;
        sum.x = sum.x * fa + y.x * fb, sum.y = sum.y * fa + y.y * fb, sum.z = sum.z * fa + y.z * fb, sum.w = sum.w * fa + y.w * fb;
    };
    bool crosses = false;
    for (int i = tid; i < runs * ROWS * V; i += kAttWorkers * 32) {
        const int run = i / (ROWS * V), r = i / V % ROWS, c = i % V * 4, p0 = run_first[run], p1 = run_last[run];
        const int4 rw = part_rows[p0];
        if (r >= rw.w) continue;
        float top = kAttFloor, den = 0.0f;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = p0; p <= p1; ++p)
            if (part_item[p][0] == part_item[p0][0])
                join(top, den, sum, P.part + (static_cast<size_t>(blockIdx.x) * P.workers * 2 + p) * kAttMaxRows * PITCH + r * PITCH, c);
        if (part_item[p0][0] >= cta0 && part_item[p0][1] <= cta1) {
            put(rw, r, c, sum, den);
        } else {
            float *to = P.cta_part + (static_cast<size_t>(blockIdx.x) * 2 + (part_item[p0][0] <= cta0 ? 0 : 1)) * kAttMaxRows * PITCH + r * PITCH;
            __stcg(reinterpret_cast<float4 *>(to + c), sum);
            if (c == 0) __stcg(reinterpret_cast<float2 *>(to + D), make_float2(top, den));
        }
    }
    // ---- and of the CTAs: the first or the last run may be shared with others
    const bool shared0 = !(part_item[run_first[0]][0] >= cta0 && part_item[run_first[0]][1] <= cta1);
    const bool shared1 = runs > 1 && !(part_item[run_first[runs - 1]][0] >= cta0 && part_item[run_first[runs - 1]][1] <= cta1);
    crosses = shared0 || shared1;
    if (!crosses) return;
    __threadfence();
    att_bar();
    if (tid < 2 && (tid == 0 ? shared0 : shared1)) {
        const int run = tid == 0 ? 0 : runs - 1;
        const int c0 = static_cast<int>(part_item[run_first[run]][0] / cta_chunk), c1 = static_cast<int>((part_item[run_first[run]][1] - 1) / cta_chunk);
        const unsigned before = atomicAdd(P.arrived + c0, 1u);
        if (before == static_cast<unsigned>(c1 - c0)) {
            P.arrived[c0] = 0u;
            last_one[tid] = run;
        }
        __threadfence();
    }
    att_bar();
    for (int w = 0; w < 2; ++w) {
        const int run = last_one[w];
        if (run < 0) continue;
        const int p0 = run_first[run];
        const long long item0 = part_item[p0][0], item1 = part_item[p0][1];
        const int c0 = static_cast<int>(item0 / cta_chunk), c1 = static_cast<int>((item1 - 1) / cta_chunk);
        const int4 rw = part_rows[p0];
        for (int i = tid; i < rw.w * V; i += kAttWorkers * 32) {
            const int r = i / V, c = i % V * 4;
            float top = kAttFloor, den = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int u = c0; u <= c1; ++u)
                join(top, den, sum, P.cta_part + (static_cast<size_t>(u) * 2 + (item0 <= u * cta_chunk ? 0 : 1)) * kAttMaxRows * PITCH + r * PITCH, c);
            put(rw, r, c, sum, den);
        }
    }
}

}  // namespace wd
