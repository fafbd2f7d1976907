// Attention over the 8-bit cache for many rows (a prompt's chunk), on the fifth-generation tensor cores. The arithmetic is that of the kernel for few
// rows (wd_kv_attend.cuh), with E = 2^(7 + x - m) and P = E 2^6 sv in F16 (hi + lo for F32 rows; for rows of 16 bits lo is left out, and the 7 are 3). A
// multiplication each is dear here (184 -> 204 us): where the value scales of a head have never been more than 2^90 apart, P is made at once as
// 2^(13 + x + log2 sv - m), and the denominator takes P 2^-6 / sv, which is E. (Farther apart P may be nothing where E is not.)
//
// An item is 128 TILES rows of one kv head of a sequence (the G query heads of a token are neighbouring rows) against the tokens that they see, KT = 128
// at a time (64 where F32 rows of 256 leave no room). Scores, then weights in their place, and sums are in tensor memory:
//
//   warps 0 .. 3, 4 .. 7   a row tile each, a thread a row: scores -> weights; the sums are brought to a new maximum only when it has grown by 2^2
//                          (16 bits: 2^6; weights stay below 2^15), then the answer at the item's end
//   warps 8 .. 11          codes -> F16 operands in shared memory, K-major without swizzle; the tokens of a sub-block are taken in the order in which a
//                          value's bytes have them, for keys and values alike
//   warp 12                issues the products, the two row tiles in turn: Q K of the next tokens, P V of these (a warp for each tile is slower:
//                          196 us with one, 209 with two)
//
// Items are dealt out heaviest first, back and forth over the CTAs (the last rows of a sequence see the most). Where there are not half as many as CTAs
// each is cut into as many runs of its tokens as fill them, and a second kernel puts the runs' sums together.
//
// Bound: heads of 64 by the softmax: the two row tiles' warps on a scheduler take about 4,400 cycles for 128 columns each, 2,048 of them the exponential
// unit's: they run nearly one after the other. 4,000 rows behind 1,011 tokens, 32 heads over 8: of 64 193 us (510 TFLOP/s; exponential pipe 52 %, tensor pipe
// 23 %), of 128 275 us (717; 37 and 33 %), of 256 893 us (442); F32 rows, with twice the products, of 64 301 us, of 128 420, of 256 1,312.
#pragma once

#include "wd_kv_attend.cuh"
#include "wd_tcgen05.cuh"

namespace wd {

constexpr int kPromptThreads = 512;
// Registers a thread: two warpgroups that work on scores take what the two others give back (128 at launch).
constexpr int kPromptRegsMore = 176, kPromptRegsLess = 80;
static_assert(2 * (kPromptRegsMore + kPromptRegsLess) <= 4 * 128, "more than the block was launched with: the increase would wait for ever");

struct KvPrompt {
    const uint8_t *pool;        // of the layer
    const float *scales;        // of the layer
    const int *book;
    const int *table;
    const int2 *reach;          // of the layer, [kv heads]
    const void *q;
    void *out;
    long long q_stride, out_stride;
    unsigned *status;
    float *part;                // [CTAs]: sums [row tile][D / 4][128 rows][4], then [rows] of maximum and denominator; until an item's end the sums of its chains
    float scale_log2;
    int type, window, vec, split, ctas;         // vec: rows of q and out lie on boundaries of 16 bytes; split: items may be cut into runs
    KvShape s;
};

template <int D, bool SPLIT>
struct PromptAttPlan {
    static constexpr int kTiles = D <= 128 ? 2 : 1, kKt = D == 256 && SPLIT ? 64 : 128, kRows = 128 * kTiles;
    static constexpr int kQ = 128 * D * 2, kQTile = kQ * (SPLIT ? 2 : 1);               // bytes: a tile's hi (or lo), both
    static constexpr int kKStep = kKt * 16, kK = D / 8 * kKStep;                        // eight elements of the head of all tokens, all of them
    static constexpr int kVStep = D * 16 + 64, kV = kKt / 8 * kVStep;                   // eight tokens of all elements (and 64 bytes, which spread the stores over the banks)
    static constexpr int kStages = kTiles * kQTile + 2 * (kK + kV) <= 216 * 1024 ? 2 : 1;
    static constexpr int kSmem = kTiles * kQTile + kStages * (kK + kV) + (kAttMaxSeqs + 4) * 4 + 1024;
    // Tensor memory: scores of each tile, then sums, then weights where there is room for them beside the scores. (Then the next scores are made while
    // a tile's weights still are.)
    static constexpr int kColO = 128 * kTiles, kColP = kColO + kTiles * D, kWidthP = kKt / 2 * (SPLIT ? 2 : 1);
    static constexpr bool kApart = kColP + kTiles * kWidthP <= 512 && kStages >= kTiles;         // (the second tile's first scores come behind the first's second)
    // Tiles after which sums are brought to memory and begun anew: a tensor core cuts its sums off, so that those of values of one sign come out low, by 3.3e-9
    // of themselves for each token and term (F32 rows, 100,000 tokens in one sum: 6.6e-4). So F32 rows add 2,048 tokens at a time, others 8,192.
    static constexpr int kChain = (SPLIT ? 2048 : 8192) / kKt;
    // The largest weight's exponent, as kAttTop, when the sums were brought to its maximum, and what it may grow by before they are again: the less, the more of
    // F16's range is there for small weights, and the more often sums are brought (4,000 rows of 64 behind 1,011 tokens: by 2^8 188 us, 2^6 192, 2^4 193).
    static constexpr float kTop = SPLIT ? 13.0f : 9.0f, kGrowth = 15.0f - kTop;
    static constexpr uint32_t kIdescS = 1u << 4 | (kKt >> 3) << 17 | (128 >> 4) << 24, kIdescO = 1u << 4 | (D >> 3) << 17 | (128 >> 4) << 24;
    static_assert(kColO + kTiles * D <= 512 && kSmem <= 226 * 1024, "plan of the memories");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Where a CTA's (or a run's) part has the four sums from column c on of a row, and its maximum and denominator: a warp's rows lie side by side.
template <int D, int ROWS>
__device__ __forceinline__ float *prompt_part(float *parts, int at, int row, int c) {
    return parts + static_cast<size_t>(at) * ROWS * (D + 4) + ((row >> 7) * (D / 4) + c / 4) * 512 + (row & 127) * 4;
}
template <int D, int ROWS>
__device__ __forceinline__ float2 *prompt_part_end(float *parts, int at, int row) {
    return reinterpret_cast<float2 *>(parts + static_cast<size_t>(at) * ROWS * (D + 4) + ROWS * D + row * 2);
}

struct PromptItem {
    int seq, row0, count, length, head, item_row, rows, lo, hi, at;         // rows: of the sequence and head; lo .. hi - 1: tiles of KT tokens; at: place of a part
};

// Items of one head in front of each sequence, and behind their number the most tiles of 128 tokens that one sees; by one warp.
__device__ __forceinline__ void prompt_prefix(const KvPrompt &P, int rows, int *prefix, int lane) {
    const int n_seq = P.book[0], g_heads = P.s.heads / P.s.kv_heads;
    const int *entries = P.book + kKvHead;
    int sum = 0, most = 0;
    for (int i0 = 0; i0 < n_seq; i0 += 32) {
        const int i = i0 + lane;
        int inc = 0;
        if (i < n_seq) {
            const int4 e = *reinterpret_cast<const int4 *>(entries + i * kKvStepWords);
            inc = static_cast<int>((static_cast<long long>(e.z) * g_heads + rows - 1) / rows);
            most = max(most, (P.window ? min(e.w, min(P.window, e.w) + rows / g_heads) : e.w) + 127 >> 7);
        }
        const int v = inc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (i < n_seq) prefix[i] = sum + inc - v;
        sum += __shfl_sync(0xffffffffu, inc, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
        prefix[n_seq] = sum;
        prefix[n_seq + 1] = most;
    }
}
// Runs that each of n items, of `most` tiles the longest, is cut into: parts and the second kernel cost what four tiles do, so that items of less than
// seven stay whole. (8 items of 63 tiles: 112 -> 27 us; of 8: 28 -> 23; 64 of 4, in two: 19 -> 33, left alone.)
__host__ __device__ inline int prompt_runs(int ctas, long long n, int most) {
    if (n < 1 || 2 * n > ctas || most < 7) return 1;
    const int fit = static_cast<int>(ctas / n), few = most / 3;
    return fit < few ? fit : few;
}
// item number n: where its rows are
__device__ __forceinline__ PromptItem prompt_item(const KvPrompt &P, const int *prefix, int n_seq, long long n, int rows) {
    PromptItem it;
    const int H = P.s.kv_heads;
    int lo = 0, hi = n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (static_cast<long long>(prefix[mid]) * H <= n) lo = mid;
        else hi = mid - 1;
    }
    const int4 e = *reinterpret_cast<const int4 *>(P.book + kKvHead + lo * kKvStepWords);
    it.seq = e.x, it.row0 = e.y, it.count = e.z, it.length = e.w;
    const int in = static_cast<int>(n - static_cast<long long>(prefix[lo]) * H), blocks = prefix[lo + 1] - prefix[lo];
    it.head = in % H;
    it.item_row = (blocks - 1 - in / H) * rows;
    it.rows = it.count * (P.s.heads / H);
    it.at = 0;
    return it;
}

template <int D, bool SPLIT, bool E4M3>
__global__ void __launch_bounds__(kPromptThreads, 1) kv_prompt_kernel(const __grid_constant__ KvPrompt P) {
    using A = PromptAttPlan<D, SPLIT>;
    constexpr int KT = A::kKt, T = A::kTiles, ST = A::kStages, CW = D % 64 == 0 ? 64 : 32, SUBS = KT / 16;
    constexpr int kPartP = A::kApart && !SPLIT ? 16 : 32;           // columns of the weights of 32 tokens
    extern __shared__ __align__(1024) uint8_t psm[];
    __shared__ __align__(8) uint64_t q_full[T], k_full[ST], k_free[ST], v_full[ST], v_free[ST], s_full[T], s_free[T], p_full[T], o_done[T];
    __shared__ __align__(16) float4 scales[4][SUBS];
    __shared__ uint32_t tmem_base;
    uint8_t *qs = psm, *ks = psm + T * A::kQTile, *vs = ks + ST * A::kK;
    int *prefix = reinterpret_cast<int *>(vs + ST * A::kV);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int n_seq = P.book[0], g_heads = P.s.heads / P.s.kv_heads, H = P.s.kv_heads;
    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < ST; ++i) {
                mbar_init(&k_full[i], 128);
                mbar_init(&v_full[i], 128);
                mbar_init(&k_free[i], 1);
                mbar_init(&v_free[i], 1);
            }
            for (int i = 0; i < T; ++i) {
                mbar_init(&s_full[i], 2);         // the products' completion, and the thread that issued them
                mbar_init(&q_full[i], 128);
                mbar_init(&s_free[i], 128);
                mbar_init(&p_full[i], 128);
                mbar_init(&o_done[i], 1);
            }
            mbar_fence_init();
        }
        prompt_prefix(P, A::kRows, prefix, lane);
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_base;
    const long long n_items = static_cast<long long>(prefix[n_seq]) * H;

    const int runs = P.split ? prompt_runs(P.ctas, n_items, prefix[n_seq + 1]) : 1;
    // item number `turn` of this CTA, or its run of one; false behind the last
    auto item_of = [&](int turn, PromptItem &it) {
        const long long at = static_cast<long long>(turn) * gridDim.x + (turn & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (at >= n_items * runs) return false;
        it = prompt_item(P, prefix, n_seq, runs > 1 ? at / runs : at, A::kRows);
        const int start = it.length - it.count, pos0 = start + it.item_row / g_heads, pos1 = start + min(it.item_row + A::kRows - 1, it.rows - 1) / g_heads;
        it.lo = P.window ? max(0, pos0 - P.window + 1) / KT : 0;
        it.hi = pos1 / KT + 1;
        if (runs > 1) {
            const int run = static_cast<int>(at % runs), n = it.hi - it.lo, lo = it.lo;
            it.lo = lo + static_cast<int>(static_cast<long long>(n) * run / runs);
            it.hi = lo + static_cast<int>(static_cast<long long>(n) * (run + 1) / runs);
            it.at = static_cast<int>(at);
        }
        return true;
    };

    PromptItem it;
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptRegsLess));
        if (warp == 12) {
            int k = 0, v = 0, items = 0;            // tiles of keys and of values that products have been issued for, items
            int n_p[2] = {0, 0}, n_f[2] = {0, 0};
            auto score = [&](int x, int i0) {       // of key tile k + i0
                const uint32_t d = tm + x * 128;
                const uint32_t q0 = smem_u32(qs + x * A::kQTile), k0 = smem_u32(ks + ((k + i0) % ST) * A::kK);
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    tc_mma_f16(d, tc_smem_desc(q0 + i * 4096, 2048), tc_smem_desc(k0 + i * 2 * A::kKStep, A::kKStep), A::kIdescS, i > 0);
                if constexpr (SPLIT) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        tc_mma_f16(d, tc_smem_desc(q0 + A::kQ + i * 4096, 2048), tc_smem_desc(k0 + i * 2 * A::kKStep, A::kKStep), A::kIdescS, 1);
                }
                tc_commit_warp(&s_full[x]);
                if (lane == 0) mbar_arrive(&s_full[x]);         // what this thread saw of the keys' warps, for those who read the scales
            };
            auto weigh = [&](int x, bool add) {     // with value tile v
                const uint32_t d = tm + A::kColO + x * D, p = tm + (A::kApart ? A::kColP + x * A::kWidthP : x * 128), v0 = smem_u32(vs + (v % ST) * A::kV);
#pragma unroll
                for (int i = 0; i < KT / 16; ++i) {
                    const uint64_t desc = tc_smem_desc(v0 + i * 2 * A::kVStep, A::kVStep);
                    tc_mma_f16_t(d, p + i / 2 * kPartP + i % 2 * 8, desc, A::kIdescO, add || i > 0);
                    if constexpr (SPLIT) tc_mma_f16_t(d, p + i / 2 * kPartP + i % 2 * 8 + 16, desc, A::kIdescO, 1);
                }
                tc_commit_warp(&o_done[x]);
                ++n_p[x];
            };
            auto keys = [&](int i) { att_wait(&k_full[(k + i) % ST], (k + i) / ST & 1, P.status); };
            // the item's first scores of a tile: the last item's have been read, or its weights, which lie where these scores go
            auto begin = [&](int x) {
                att_wait(&q_full[x], items & 1, P.status);
                if (A::kApart && n_p[x] > 0) att_wait(&s_free[x], n_f[x]++ & 1, P.status);
                if (!A::kApart && n_p[x] > 0) att_wait(&o_done[x], (n_p[x] - 1) & 1, P.status);
                tc_fence_after();
                score(x, 0);
            };
            auto weights = [&](int x, int j) {
                att_wait(&p_full[x], n_p[x] & 1, P.status);
                tc_fence_after();
                weigh(x, j % A::kChain != 0);
            };
            for (int turn = 0; item_of(turn, it); ++turn, ++items) {
                const int n = it.hi - it.lo;
                if (n == 0) break;              // (a run of a short item; there is no other item then)
                keys(0);
                if constexpr (A::kApart && T == 2) {
                    // The second tile begins when the first has its weights, and stays that much behind: one makes exponentials while the other reads
                    // scores and looks for their maximum.
                    begin(0);
                    for (int j = 0; j < n; ++j, ++k, ++v) {
                        if (j + 1 < n) {
                            keys(1);
                            att_wait(&s_free[0], n_f[0]++ & 1, P.status);
                            tc_fence_after();
                            score(0, 1);
                        }
                        att_wait(&v_full[v % ST], v / ST & 1, P.status);
                        weights(0, j);
                        if (j == 0) {
                            begin(1);
                            tc_commit_warp(&k_free[k % ST]);
                        }
                        if (j + 1 < n) {
                            att_wait(&s_free[1], n_f[1]++ & 1, P.status);
                            tc_fence_after();
                            score(1, 1);
                            tc_commit_warp(&k_free[(k + 1) % ST]);
                        }
                        weights(1, j);
                        tc_commit_warp(&v_free[v % ST]);
                    }
                } else {
                    for (int x = 0; x < T; ++x) begin(x);
                    tc_commit_warp(&k_free[k % ST]);
                    for (int j = 0; j < n; ++j, ++k, ++v) {
                        if (j + 1 < n) keys(1);
                        if (A::kApart && j + 1 < n) {
                            for (int x = 0; x < T; ++x) {
                                att_wait(&s_free[x], n_f[x]++ & 1, P.status);
                                tc_fence_after();
                                score(x, 1);
                            }
                            tc_commit_warp(&k_free[(k + 1) % ST]);
                        }
                        att_wait(&v_full[v % ST], v / ST & 1, P.status);
                        for (int x = 0; x < T; ++x) {
                            weights(x, j);
                            if (x == T - 1) tc_commit_warp(&v_free[v % ST]);
                            if (!A::kApart && j + 1 < n) {
                                att_wait(&o_done[x], (n_p[x] - 1) & 1, P.status);
                                tc_fence_after();
                                score(x, 1);
                                if (x == T - 1) tc_commit_warp(&k_free[(k + 1) % ST]);
                            }
                        }
                    }
                }
            }
            for (int x = 0; x < T; ++x)
                if (n_p[x] > 0) tc_drain(&o_done[x], (n_p[x] - 1) & 1);
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptRegsLess));
        const int ct = tid - 256, cw = warp - 8, shift = P.s.page_shift;
        int n = 0;              // tiles so far
        for (int turn = 0; item_of(turn, it); ++turn) {
            const int *table = P.table + static_cast<size_t>(it.seq) * P.s.max_pages;
            const int last_sub = (it.length - 1) >> 4;
            const uint8_t *head = P.pool + it.head * kv_head_bytes(P.s);
            const float zero = kv_zero_scale(P.reach[it.head]);        // what stands for a scale of 0
            // lane l: page of sub-block l of a tile, where the sub-block is in the page, and the scales (behind the last sub-block: the last one)
            int page = 0, in_page = 0;
            float2 sc = make_float2(0.0f, 0.0f);
            auto look_up = [&](int tile) {
                const int sub = min(tile * SUBS + (lane & (SUBS - 1)), last_sub);
                page = table[sub >> (shift - 4)];
                in_page = sub & ((1 << (shift - 4)) - 1);
                if (cw == 0) sc = *reinterpret_cast<const float2 *>(P.scales + (static_cast<size_t>(page) * H + it.head) * 2);
            };
            if (it.lo < it.hi) look_up(it.lo);
            for (int tile = it.lo; tile < it.hi; ++tile, ++n) {
                const size_t at = static_cast<size_t>(page) * kv_page_bytes(P.s) + static_cast<size_t>(in_page) * (16 * D);
                const float vsc = sc.y > 0.0f ? sc.y : zero, up = static_cast<float>(1 << kAttScale);
                const float4 mine = make_float4(sc.x, log2f(vsc), 1.0f / (up * vsc), up * sc.y);
                const int st = n % ST;
                const uint32_t par = (static_cast<uint32_t>(n / ST) & 1u) ^ 1u;
                // keys: unit u is 16 elements of token u % KT
                constexpr int KU = KT * D / 16 / 128, KB = KU < 8 ? KU : 8;
                const int row = ct % KT, sub = row >> 4, place = row & 15, token = (place >> 2) * 2 + (place & 1) + ((place & 2) << 2);
                const uint8_t *kp = head + __shfl_sync(0xffffffffu, at, sub) + token * CW;
                auto key_at = [&](int i) {
                    const int k16 = (i * 128 + ct) / KT * 16;
                    return reinterpret_cast<const uint4 *>(kp + k16 / CW * (16 * CW) + k16 % CW);
                };
                // values: a warp takes 512 bytes (16 tokens of 32 elements) at a time
                constexpr int VU = SUBS * (D / 32) / 4, VB = VU < 8 ? VU : 8;
                constexpr bool kBoth = KU <= 4 && VU <= 4;         // both asked for at once, where the registers hold them
                auto value_at = [&](int i) {
                    const int u = i * 4 + cw, s = u / (D / 32), blk = u % (D / 32);
                    return reinterpret_cast<const uint4 *>(head + __shfl_sync(0xffffffffu, at, s) + kv_half_bytes(P.s) + blk * 512 + lane * 16);
                };
                uint4 raw[KB], val[VB];
#pragma unroll
                for (int i = 0; i < KB; ++i) raw[i] = __ldg(key_at(i));
                if constexpr (kBoth) {
#pragma unroll
                    for (int i = 0; i < VB; ++i) val[i] = __ldg(value_at(i));
                }
                att_wait(&k_free[st], par, P.status);
#pragma unroll
                for (int b = 0; b < KU; b += KB) {
                    if (b > 0) {
#pragma unroll
                        for (int i = 0; i < KB; ++i) raw[i] = __ldg(key_at(b + i));
                    }
#pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        const int k16 = ((b + i) * 128 + ct) / KT;
                        uint4 *to = reinterpret_cast<uint4 *>(ks + st * A::kK + k16 * 2 * A::kKStep + row * 16);
                        uint4 lo, hi;
                        kv_halves<E4M3>(raw[i].x, lo.x, lo.y);
                        kv_halves<E4M3>(raw[i].y, lo.z, lo.w);
                        kv_halves<E4M3>(raw[i].z, hi.x, hi.y);
                        kv_halves<E4M3>(raw[i].w, hi.z, hi.w);
                        to[0] = lo;
                        to[A::kKStep / 16] = hi;
                    }
                }
                if (cw == 0 && lane < SUBS) scales[n & 3][lane] = mine;
                fence_proxy_async();
                mbar_arrive(&k_full[st]);
                if constexpr (!kBoth) {
#pragma unroll
                    for (int i = 0; i < VB; ++i) val[i] = __ldg(value_at(i));
                }
                if (tile + 1 < it.hi) look_up(tile + 1);
                att_wait(&v_free[st], par, P.status);
                const int g = lane >> 2, t = lane & 3;
#pragma unroll
                for (int b = 0; b < VU; b += VB) {
                    if (b > 0) {
#pragma unroll
                        for (int i = 0; i < VB; ++i) val[i] = __ldg(value_at(b + i));
                    }
#pragma unroll
                    for (int i = 0; i < VB; ++i) {
                        const int u = (b + i) * 4 + cw, s = u / (D / 32), blk = u % (D / 32);
                        uint8_t *to = vs + st * A::kV + (2 * s + (t >> 1)) * A::kVStep + (blk * 32 + g) * 16 + (t & 1) * 8;
                        const uint32_t w[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint2 h;
                            kv_halves<E4M3>(w[j], h.x, h.y);
                            *reinterpret_cast<uint2 *>(to + j * 128) = h;
                        }
                    }
                }
                fence_proxy_async();
                mbar_arrive(&v_full[st]);
            }
        }
    } else if (warp < 4 * T) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptRegsMore));
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lanes = tm + (static_cast<uint32_t>((warp & 3) * 32) << 16), sc = lanes + x * 128, oc = lanes + A::kColO + x * D, pc = A::kApart ? lanes + A::kColP + x * A::kWidthP : sc;
        int n_s = 0, n_o = 0, n = 0;
        for (int turn = 0; item_of(turn, it); ++turn) {
            const int row = it.item_row + x * 128 + r, last = it.rows - 1, start = it.length - it.count;
            const int pos = start + min(row, last) / g_heads;
            const int warp_row = it.item_row + x * 128 + (warp & 3) * 32, pos_lo = start + min(warp_row, last) / g_heads, pos_hi = start + min(warp_row + 31, last) / g_heads;
            const bool is = row <= last;
            const size_t elem = (static_cast<size_t>(it.head) * g_heads + row % g_heads) * D;
            const size_t src = static_cast<size_t>(it.row0 + row / g_heads) * P.q_stride + elem;
            // q: the row's largest magnitude, then its F16 terms; element k of row r lies at (k / 8) 2048 + r 16
            auto load16 = [&](int k, float *y) {
                if (!is) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = 0.0f;
                } else if (P.type == kRowsF32) {
                    row_load16(static_cast<const float *>(P.q) + src + k, P.vec != 0, y);
                } else if (P.type == kRowsF16) {
                    row_load16(static_cast<const __half *>(P.q) + src + k, P.vec != 0, y);
                } else {
                    row_load16(static_cast<const __nv_bfloat16 *>(P.q) + src + k, P.vec != 0, y);
                }
            };
            float top = 0.0f;
#pragma unroll 1
            for (int k = 0; k < D; k += 16) {
                float y[16];
                load16(k, y);
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(y[i]));
            }
            const int e = top > 0.0f ? max(-100, min(128, static_cast<int>(__float_as_uint(top) >> 23) - 126)) - 15 : 0, e1 = e / 2, e2 = e - e1;
            const float mul = P.scale_log2 * __uint_as_float((127 + e1) << 23) * __uint_as_float((127 + e2) << 23);
            const float down = __uint_as_float((127 - e1) << 23), down2 = __uint_as_float((127 - e2) << 23);
            uint8_t *to = qs + x * A::kQTile + r * 16;
#pragma unroll 1
            for (int k = 0; k < D; k += 16) {
                float y[16];
                load16(k, y);
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = y[2 * i] * down * down2, b = y[2 * i + 1] * down * down2;
                    hi[i] = half_pair(a, b);
                    if constexpr (SPLIT) lo[i] = half_rest(a, b, hi[i]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    *reinterpret_cast<uint4 *>(to + (k / 8 + i) * 2048) = make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
                    if constexpr (SPLIT) *reinterpret_cast<uint4 *>(to + A::kQ + (k / 8 + i) * 2048) = make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
                }
            }
            fence_proxy_async();
            if (it.lo < it.hi) mbar_arrive(&q_full[x]);
            float m = kAttFloor, l = 0.0f;
            // the row's maximum is now `most` or what it was; brought to it where it has grown enough
            auto follow = [&](int tile, float most) {
                if (tile == it.lo) {
                    m = most;
                } else if (__any_sync(0xffffffffu, most > m + A::kGrowth)) {
                    const float now = fmaxf(m, most), half_way = ex2(0.5f * (m - now)), f = half_way * half_way;        // (see the kernel for few rows)
                    m = now;
                    l = l * half_way * half_way;
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t u[16];
                        tc_ld(oc + c * 16, u);
                        tc_wait_ld(u);
#pragma unroll
                        for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * f);
                        tc_st(oc + c * 16, u);
                    }
                }
            };
            auto tiles = [&](auto apart) {
                constexpr bool kFar = decltype(apart)::value;
#pragma unroll 1
                for (int tile = it.lo; tile < it.hi;) {
                    const int chain_end = min(tile + A::kChain, it.hi);
#pragma unroll 1
                    for (; tile < chain_end; ++tile, ++n) {
                        att_wait(&s_full[x], n_s++ & 1, P.status);
                        tc_fence_after();
                        const int first = tile * KT;
                        const bool edge = first + KT - 1 > pos_lo || (P.window && first <= pos_hi - P.window);
                        if constexpr (kFar) {           // (rare: little code, few registers, the scores read twice)
                            float most = kAttFloor;
                            uint32_t u[32], hi[16], lo[16];
                            auto scores = [&](int c) {          // of the 32 tokens from 32 c on
                                tc_ld(sc + c * 32, u);
                                tc_wait_ld(u);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const int p = i & 15, token = first + c * 32 + (i & 16) + (p >> 2) * 2 + (p & 1) + ((p & 2) << 2);
                                    if (token > pos || (P.window && token <= pos - P.window)) u[i] = 0xff800000u;
                                }
                            };
#pragma unroll 1
                            for (int c = 0; c < KT / 32; ++c) {
                                scores(c);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float4 s4 = scales[n & 3][2 * c + i / 16];
                                    most = fmaxf(most, fmaf(__uint_as_float(u[i]), fmaxf(mul * s4.x, 1e-37f), s4.y));
                                }
                            }
                            if constexpr (A::kApart) {
                                if (n_o > 0) att_wait(&o_done[x], (n_o - 1) & 1, P.status);
                                tc_fence_after();
                            }
                            follow(tile, most);
                            const float off = (A::kTop - static_cast<float>(kAttScale)) - m;
#pragma unroll 1
                            for (int c = 0; c < KT / 32; ++c) {
                                scores(c);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const float4 s4 = scales[n & 3][2 * c + i / 8];
                                    const float mk = fmaxf(mul * s4.x, 1e-37f), a = ex2(fmaf(__uint_as_float(u[2 * i]), mk, off)), b = ex2(fmaf(__uint_as_float(u[2 * i + 1]), mk, off));
                                    l += a + b;
                                    hi[i] = half_pair(a * s4.w, b * s4.w);
                                    if constexpr (SPLIT) lo[i] = half_rest(a * s4.w, b * s4.w, hi[i]);
                                }
                                tc_st(pc + c * kPartP, hi);
                                if constexpr (SPLIT) tc_st(pc + c * kPartP + 16, lo);
                            }
                            if constexpr (A::kApart) {
                                tc_fence_before();
                                mbar_arrive(&s_free[x]);
                            }
                        } else {
                            uint32_t v[KT / 32][32];
#pragma unroll
                            for (int c = 0; c < KT / 32; ++c) tc_ld(sc + c * 32, v[c]);
#pragma unroll
                            for (int c = 0; c < KT / 32; ++c) tc_wait_ld(v[c]);
                            if constexpr (A::kApart) {
                                tc_fence_before();
                                mbar_arrive(&s_free[x]);
                            }
                            // column 16 s + p of the scores is token 2 (p / 4) + (p & 1) + 8 ((p & 3) / 2) of sub-block s
                            if (edge) {
#pragma unroll
                                for (int c = 0; c < KT / 32; ++c)
#pragma unroll
                                    for (int i = 0; i < 32; ++i) {
                                        const int p = i & 15, token = first + c * 32 + (i & 16) + (p >> 2) * 2 + (p & 1) + ((p & 2) << 2);
                                        if (token > pos || (P.window && token <= pos - P.window)) v[c][i] = 0xff800000u;
                                    }
                            }
                            float most = kAttFloor;
#pragma unroll
                            for (int b = 0; b < SUBS; ++b) {
                                const float4 s4 = scales[n & 3][b];
                                auto at = [&](int i) { return __uint_as_float(v[b / 2][b % 2 * 16 + i]); };
                                float t = max3(at(0), at(1), at(2));
#pragma unroll
                                for (int i = 3; i < 15; i += 2) t = max3(t, at(i), at(i + 1));
                                t = fmaxf(t, at(15));
                                most = fmaxf(most, fmaf(t, fmaxf(mul * s4.x, 1e-37f), s4.y));
                            }
                            if constexpr (A::kApart) {          // the sums, and the place of the weights, are free
                                if (n_o > 0) att_wait(&o_done[x], (n_o - 1) & 1, P.status);
                                tc_fence_after();
                            }
                            follow(tile, most);
                            const float base = m - A::kTop;
                            // exponents of all columns, then the exponentials (scales read between the stores of weights would wait for them)
#pragma unroll
                            for (int b = 0; b < SUBS; ++b) {
                                const float4 s4 = scales[n & 3][b];
                                const float mk = fmaxf(mul * s4.x, 1e-37f), off = s4.y - base;
                                const f32x2 mk2 = pack2(mk, mk), off2 = pack2(off, off);
#pragma unroll
                                for (int i = 0; i < 16; i += 2) {
                                    uint32_t *u = &v[b / 2][b % 2 * 16 + i];
                                    float a, c;
                                    unpack2(fma2(pack2(__uint_as_float(u[0]), __uint_as_float(u[1])), mk2, off2), a, c);
                                    u[0] = __float_as_uint(a), u[1] = __float_as_uint(c);
                                }
                            }
                            uint32_t hi[KT / 32][16], lo[SPLIT ? KT / 32 : 1][16];
#pragma unroll
                            for (int b = 0; b < SUBS; ++b) {
                                f32x2 s0 = pack2(0.0f, 0.0f), s1 = s0;
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float a = ex2(__uint_as_float(v[b / 2][b % 2 * 16 + 2 * i])), c = ex2(__uint_as_float(v[b / 2][b % 2 * 16 + 2 * i + 1]));
                                    if (i & 1) s1 = add2(s1, pack2(a, c));
                                    else s0 = add2(s0, pack2(a, c));
                                    hi[b / 2][b % 2 * 8 + i] = half_pair(a, c);
                                    if constexpr (SPLIT) lo[b / 2][b % 2 * 8 + i] = half_rest(a, c, hi[b / 2][b % 2 * 8 + i]);
                                }
                                float a, c;
                                unpack2(add2(s0, s1), a, c);
                                l = fmaf(a + c, scales[n & 3][b].z, l);
                            }
#pragma unroll
                            for (int c = 0; c < KT / 32; ++c) {
                                tc_st(pc + c * kPartP, hi[c]);
                                if constexpr (SPLIT) tc_st(pc + c * kPartP + 16, lo[c]);
                            }
                        }
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(&p_full[x]);
                        ++n_o;
                    }
                    // a chain's end: its sums are added to those of the chains in front of it
                    if (tile < it.hi) {
                        int of = x * 128 + r;
                        asm volatile("" : "+r"(of));          // (addresses are made here, not held through the tiles)
                        const int place = runs > 1 ? it.at : blockIdx.x;
                        const bool more = tile - it.lo > A::kChain;
                        float *held_m = &prompt_part_end<D, A::kRows>(P.part, place, of)->x;
                        const float f = more ? ex2(*held_m - m) : 0.0f;         // (m does not go down)
                        *held_m = m;
                        float4 h[8];
                        auto ask = [&](int c) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) h[i] = more ? *reinterpret_cast<const float4 *>(prompt_part<D, A::kRows>(P.part, place, of, c + 4 * i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        };
                        ask(0);
                        att_wait(&o_done[x], (n_o - 1) & 1, P.status);
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t u[32];
                            tc_ld(oc + c, u);
                            tc_wait_ld(u);
                            float4 y[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                y[i] = make_float4(fmaf(h[i].x, f, __uint_as_float(u[4 * i])), fmaf(h[i].y, f, __uint_as_float(u[4 * i + 1])),
                                                   fmaf(h[i].z, f, __uint_as_float(u[4 * i + 2])), fmaf(h[i].w, f, __uint_as_float(u[4 * i + 3])));
                            if (c + 32 < D) ask(c + 32);
#pragma unroll
                            for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(prompt_part<D, A::kRows>(P.part, place, of, c + 4 * i)) = y[i];
                        }
                        tc_fence_before();
                    }
                }
            };
            if (kv_far_apart(P.reach[it.head])) tiles(std::true_type{});
            else tiles(std::false_type{});
            if (it.lo < it.hi) att_wait(&o_done[x], (n_o - 1) & 1, P.status);
            tc_fence_after();
            const bool held = it.hi - it.lo > A::kChain;
            int of = x * 128 + r;
            asm volatile("" : "+r"(of));
            const int place = runs > 1 ? it.at : blockIdx.x;
            const float f_held = held ? ex2(prompt_part_end<D, A::kRows>(P.part, place, of)->x - m) : 0.0f;
            // 16 columns of the sums
            auto sums = [&](int c, uint32_t (&v)[16]) {
                tc_ld(oc + c * 16, v);
                tc_wait_ld(v);
                if (held) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 h = *reinterpret_cast<const float4 *>(prompt_part<D, A::kRows>(P.part, place, of, c * 16 + i));
                        v[i] = __float_as_uint(fmaf(h.x, f_held, __uint_as_float(v[i])));
                        v[i + 1] = __float_as_uint(fmaf(h.y, f_held, __uint_as_float(v[i + 1])));
                        v[i + 2] = __float_as_uint(fmaf(h.z, f_held, __uint_as_float(v[i + 2])));
                        v[i + 3] = __float_as_uint(fmaf(h.w, f_held, __uint_as_float(v[i + 3])));
                    }
                }
            };
            if (runs > 1) {         // for the kernel behind
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t v[16];
                    sums(c, v);
                    if (is && it.lo < it.hi) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *reinterpret_cast<uint4 *>(prompt_part<D, A::kRows>(P.part, place, of, c * 16 + i)) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
                    __syncwarp();
                }
                if (is) *prompt_part_end<D, A::kRows>(P.part, place, of) = make_float2(m, l);         // (of an empty run nothing else is read)
                continue;
            }
            const float inv = kAttUnit / l;
            const size_t dst = static_cast<size_t>(it.row0 + row / g_heads) * P.out_stride + elem;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
                uint32_t v[16];
                sums(c, v);
                if (is) {
                    float y[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(v[i]) * inv;
                    auto put = [&](auto *o) {
                        using R = std::remove_pointer_t<decltype(o)>;
                        __align__(16) R z[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[i] = row_number<R>(y[i]);
                        if (P.vec) {
#pragma unroll
                            for (int i = 0; i < static_cast<int>(sizeof(z)) / 16; ++i) reinterpret_cast<uint4 *>(o)[i] = reinterpret_cast<const uint4 *>(z)[i];
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = z[i];
                        }
                    };
                    if (P.type == kRowsF32) put(static_cast<float *>(P.out) + dst + c * 16);
                    else if (P.type == kRowsF16) put(static_cast<__half *>(P.out) + dst + c * 16);
                    else put(static_cast<__nv_bfloat16 *>(P.out) + dst + c * 16);
                }
                __syncwarp();
            }
            tc_fence_before();      // the sums have been read: the next item's may be written once its weights are there
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptRegsMore));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
}

// The runs' sums of each row of the items: a thread has four elements of a row, a warp 32 rows.
template <int D>
__global__ void __launch_bounds__(256) kv_prompt_join_kernel(const __grid_constant__ KvPrompt P) {
    constexpr int ROWS = D <= 128 ? 256 : 128, UNITS = ROWS * (D / 4);
    __shared__ int prefix[kAttMaxSeqs + 2];
    const int tid = threadIdx.x, n_seq = P.book[0], g_heads = P.s.heads / P.s.kv_heads;
    if (tid < 32) prompt_prefix(P, ROWS, prefix, tid);
    __syncthreads();
    const long long n_items = static_cast<long long>(prefix[n_seq]) * P.s.kv_heads;
    const int runs = P.split ? prompt_runs(P.ctas, n_items, prefix[n_seq + 1]) : 1;
    if (runs == 1) return;
    for (long long u = static_cast<long long>(blockIdx.x) * 256 + tid; u < n_items * UNITS; u += static_cast<long long>(gridDim.x) * 256) {
        const long long n = u / UNITS;
        const int in = static_cast<int>(u % UNITS), r = in % ROWS, c = in / ROWS * 4;
        const PromptItem it = prompt_item(P, prefix, n_seq, n, ROWS);
        const int row = it.item_row + r;
        if (row >= it.rows) continue;
        const int at = static_cast<int>(n) * runs;
        float top = kAttFloor, den = 0.0f;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = 0; k < runs; ++k) top = fmaxf(top, prompt_part_end<D, ROWS>(P.part, at + k, r)->x);
#pragma unroll 4
        for (int k = 0; k < runs; ++k) {
            const float2 z = *prompt_part_end<D, ROWS>(P.part, at + k, r);
            const float4 y = *reinterpret_cast<const float4 *>(prompt_part<D, ROWS>(P.part, at + k, r, c));
            if (z.y == 0.0f) continue;          // (an empty run has no sums)
            const float half_way = ex2(0.5f * (z.x - top)), f = half_way * half_way;
            den += z.y * half_way * half_way;
            sum.x = fmaf(y.x, f, sum.x), sum.y = fmaf(y.y, f, sum.y), sum.z = fmaf(y.z, f, sum.z), sum.w = fmaf(y.w, f, sum.w);
        }
        const float inv = kAttUnit / den;
        const size_t to = static_cast<size_t>(it.row0 + row / g_heads) * P.out_stride + (static_cast<size_t>(it.head) * g_heads + row % g_heads) * D + c;
        row_store(P.out, P.type, to, sum.x * inv);
        row_store(P.out, P.type, to + 1, sum.y * inv);
        row_store(P.out, P.type, to + 2, sum.z * inv);
        row_store(P.out, P.type, to + 3, sum.w * inv);
    }
}

}  // namespace wd
