// Attention over the 8-bit cache for trees of drafted tokens, on the fifth-generation tensor cores. The arithmetic is that of the kernel for prompts
// (wd_kv_prompt.cuh); which of the step's tokens a row sees is looked up on its way to the root, where a tile reaches into the step.
//
// A tree has few rows and a long context: an item is 128 rows of one kv head of a sequence (the G query heads of a token are neighbouring rows) against all
// tokens that the sequence's rows see, KT = 128 at a time, 64 of F32 rows of 128, 32 of 256: so that there is room for two stages of operands and a tile of
// codes on its way (F32 rows of 128, 131,000 tokens: 430 us by 128 with the codes read when they are needed, 289 by 64; of 256 631 and 463). All items' tiles are numbered through and each CTA takes an
// equal run of the numbers, whatever the sequences' lengths; a second kernel puts together the items that several CTAs have a part of (by the last CTA that brings one it took
// 17 us for nine parts of heads of 128, by all SMs 5).
//
//   warps 0 .. 3, 4 .. 7   a thread a row: scores -> weights. Both have the same rows: one takes the even tiles, the other the odd ones, each with sums and a
//                          maximum of its own, which are put together at the item's end (heads of 256: the first alone, tensor memory has no room for two)
//   warps 8 .. 11          codes -> F16 operands in shared memory (keys by four warps and values by three is slower, 1.4 us a tile of heads of 64 for 1.25: the
//                          warps that work on scores get fewer issue slots)
//   warp 12                issues the products
//
// A CTA's parts in memory are three units of 128 rows: what it has of an item that began in an earlier one's run; and the sums of the two streams until an
// item's end, the first of which then holds what it has of an item that ends in a later one's.
//
// A tile of 128 rows by 128 tokens takes a CTA 1.75 us at heads of 128, 1.1 at 64. 16 trees of 26 rows behind 300 to 6,000 tokens, 32/8 heads of 128: 64 us (12 at the memory's
// rate; by the kernel of chains 145), of which the beginnings and ends of items are as much as their tiles: latency, with issue slots 29 % busy, tensor cores 17 %, the exponentials' unit
// 18 %, DRAM 17 %, and stalls on memory (35 %) and at the barriers between an item's parts (27 %); 64 rows behind 131,025: 207 to 233 (83 at the tensor cores' rate). There
// both row blocks of a head expand the same codes, which the kernel for prompts does once for 256 rows (184): choose_tree() gives it such steps.
#pragma once

#include "wd_kv_prompt.cuh"

namespace wd {

struct KvTree : KvPrompt {
    const int *parents;         // see KvAttendTree
    int4 *cuts;                 // [CTAs][2]: of the item that begins in a CTA's run and ends behind it: its sequence's first row, rows of a head, head, first row; CTA of its end (-1: none)
};

template <int D, bool SPLIT>
struct TreePlan {
    static constexpr int kStreams = D <= 128 ? 2 : 1, kKt = D == 256 ? 32 : D == 128 && SPLIT ? 64 : 128;
    static constexpr int kQ = 128 * D * 2, kQTile = kQ * (SPLIT ? 2 : 1);
    static constexpr int kKStep = kKt * 16, kK = D / 8 * kKStep, kVStep = D * 16 + 64, kV = kKt / 8 * kVStep;
    static constexpr int kCodes = 2 * kKt * D, kFit = (209 * 1024 - kQTile - kCodes) / (kK + kV), kStages = kFit > 4 ? 4 : kFit;        // a tile's codes on their way; stages of operands
    static constexpr int kSmem = kQTile + kStages * (kK + kV) + kCodes + (kAttMaxSeqs + 2) * 8 + kAttEntries * 16 + 1024;
    static constexpr int kColO = 128 * kStreams, kColP = kColO + kStreams * D, kWidthP = kKt / 2 * (SPLIT ? 2 : 1);
    static constexpr bool kApart = kColP + kStreams * kWidthP <= 512;
    static constexpr int kChain = (SPLIT ? 2048 : 8192) / kKt;          // tiles of a stream
    static constexpr float kTop = SPLIT ? 13.0f : 9.0f, kGrowth = 15.0f - kTop;
    static constexpr uint32_t kIdescS = 1u << 4 | (kKt >> 3) << 17 | (128 >> 4) << 24, kIdescO = 1u << 4 | (D >> 3) << 17 | (128 >> 4) << 24;
    static constexpr int kScales = 8;       // tiles whose scales are held: a stage is free four tiles behind the softmax at most
    static_assert(kColO + kStreams * D <= 512 && kStages >= 2 && kSmem <= 220 * 1024, "plan of the memories");
};
// Tiles that every item of a sequence has.
__host__ __device__ inline int tree_first_tile(int length, int count, int window, int kt) {
    const int first = length - count - window + 1;
    return window && first > 0 ? first / kt : 0;
}
__host__ __device__ inline int tree_tiles(int length, int count, int window, int kt) { return (length + kt - 1) / kt - tree_first_tile(length, count, window, kt); }
// The run of a CTA: two tiles of 128 tokens at least (1,000 tokens, 60 rows of 4 x 64: by four 17.1 us, by two 15.9).
__host__ __device__ inline long long tree_chunk(long long total, int ctas, int most, int kt) {
    const long long even = total < (1ll << 31) ? static_cast<long long>((static_cast<uint32_t>(total) + ctas - 1) / static_cast<uint32_t>(ctas)) : (total + ctas - 1) / ctas, least = 256 / kt < most ? 256 / kt : most;
    return even > least ? even : least;
}

// An item counts a few tiles more than it has, in front of them, for what it costs to begin and end one.
constexpr int kTreeExtra = 6;

struct TreeSegment {
    int seq, row0, count, length, head, item_row, rows, lo, hi;     // rows: of the sequence and head; lo .. hi - 1: tiles of KT tokens
    bool whole, begun;          // it holds all of the item; the item began in an earlier CTA's run
    long long tile0, tile1, next;       // numbers: of the item's tiles; the one behind the segment
};
// Numbers of one head in front of each sequence; behind their number that of the tiles that an item has at most. By one warp.
__device__ __forceinline__ void tree_prefix(const KvTree &P, int kt, long long *prefix, int4 *step, int lane) {
    const int n_seq = P.book[0], g_heads = P.s.heads / P.s.kv_heads;
    const int *entries = P.book + kKvHead;
    long long sum = 0;
    int most = 0, most_rows = 0;
    for (int i0 = 0; i0 < n_seq; i0 += 32) {
        const int i = i0 + lane;
        long long inc = 0;
        if (i < n_seq) {
            const int4 e = *reinterpret_cast<const int4 *>(entries + i * kKvStepWords);
            if (i < kAttEntries) step[i] = e;
            const int n = e.z > 0 ? tree_tiles(e.w, e.z, P.window, kt) : 0;
            inc = static_cast<long long>((e.z * g_heads + 127) / 128) * (n + kTreeExtra);
            most = max(most, n);
            most_rows = max(most_rows, e.z);
        }
        const long long v = inc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (i < n_seq) prefix[i] = sum + inc - v;
        sum += __shfl_sync(0xffffffffu, inc, 31);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (__any_sync(0xffffffffu, most_rows > kTreeRows)) sum = 0;        // (a replay on such a step does nothing)
    if (lane == 0) {
        prefix[n_seq] = sum;
        prefix[n_seq + 1] = most;
    }
}
// the segment of the numbers at .. end - 1 that belongs to one item (lo == hi where it has none of its tiles); `begin`: of the CTA's run
__device__ __forceinline__ TreeSegment tree_segment(const KvTree &P, int kt, const long long *prefix, const int4 *step, int n_seq, long long begin, long long at, long long end) {
    TreeSegment s;
    const int H = P.s.kv_heads;
    int lo = 0, hi = n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] * H <= at) lo = mid;
        else hi = mid - 1;
    }
    const int4 e = lo < kAttEntries ? step[lo] : *reinterpret_cast<const int4 *>(P.book + kKvHead + lo * kKvStepWords);
    s.seq = e.x, s.row0 = e.y, s.count = e.z, s.length = e.w;
    const int tiles = tree_tiles(s.length, s.count, P.window, kt), first = tree_first_tile(s.length, s.count, P.window, kt);
    const uint32_t per = tiles + kTreeExtra, g_heads = P.s.heads / H, blocks = (s.count * g_heads + 127) / 128;
    const long long in = at - prefix[lo] * H;
    // (numbers that 32 bits hold are divided in 32 bits; there are fewer items than rows of heads, which 32 bits count)
    const uint32_t item = in < (1ll << 31) ? static_cast<uint32_t>(in) / per : static_cast<uint32_t>(in / per);
    s.head = static_cast<int>(item / blocks);
    s.item_row = static_cast<int>(item % blocks) * 128;
    s.rows = s.count * g_heads;
    s.tile0 = prefix[lo] * H + static_cast<long long>(item) * per + kTreeExtra;
    s.tile1 = s.tile0 + tiles;
    s.next = min(s.tile1, end);
    s.lo = first + static_cast<int>(max(at, s.tile0) - s.tile0);
    s.hi = max(s.lo, first + static_cast<int>(s.next - s.tile0));
    s.whole = s.hi - s.lo == tiles;
    s.begun = s.tile0 < begin;
    return s;
}

template <int D, bool SPLIT, bool E4M3>
__global__ void __launch_bounds__(kPromptThreads, 1) kv_tree_kernel(const __grid_constant__ KvTree P) {
    using A = TreePlan<D, SPLIT>;
    constexpr int KT = A::kKt, X = A::kStreams, ST = A::kStages, CW = D % 64 == 0 ? 64 : 32, SUBS = KT / 16;
    constexpr int kPartP = A::kApart && !SPLIT ? 16 : 32;           // columns of the weights of 32 tokens
    extern __shared__ __align__(1024) uint8_t tsm[];
    __shared__ __align__(8) uint64_t q_full, k_full[ST], k_free[ST], v_full[ST], v_free[ST], s_full[X], s_free[X], p_full[X], o_done[X];
    __shared__ __align__(16) float4 scales[A::kScales][SUBS], ends[X][128];
    __shared__ float muls[128];            // of a row's scores, what its terms were divided by too
    __shared__ int8_t places[2][kTreeRows];         // parents of a segment's rows, and of the one's behind it
    __shared__ uint32_t tmem_base;
    uint8_t *qs = tsm, *ks = tsm + A::kQTile, *vs = ks + ST * A::kK, *raws = vs + ST * A::kV;
    int4 *step = reinterpret_cast<int4 *>(raws + A::kCodes);            // the first entries of the step
    long long *prefix = reinterpret_cast<long long *>(step + kAttEntries);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int n_seq = P.book[0], g_heads = P.s.heads / P.s.kv_heads, H = P.s.kv_heads;
    if (warp == 0) {
        if (lane == 0) {
            mbar_init(&q_full, 128 * X);
            for (int i = 0; i < ST; ++i) {
                mbar_init(&k_full[i], 128);
                mbar_init(&v_full[i], 128);
                mbar_init(&k_free[i], 1);
                mbar_init(&v_free[i], 1);
            }
            for (int i = 0; i < X; ++i) {
                mbar_init(&s_full[i], 2);         // the products' completion, and the thread that issued them
                mbar_init(&s_free[i], 128);
                mbar_init(&p_full[i], 128);
                mbar_init(&o_done[i], 1);
            }
            mbar_fence_init();
        }
        tree_prefix(P, KT, prefix, step, lane);
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_base;
    // This CTA's numbers; or whole items, in turn.
    const long long total = prefix[n_seq] * H, chunk = P.split ? tree_chunk(total, gridDim.x, static_cast<int>(prefix[n_seq + 1]), KT) : 0;
    const long long begin = min(blockIdx.x * chunk, total), end = min(begin + chunk, total);
    // the segment behind `at` (-1: the first one); false behind the last
    auto next_segment = [&](long long &at, TreeSegment &s) {
        if (P.split) {
            for (at = at < 0 ? begin : at; at < end;) {
                s = tree_segment(P, KT, prefix, step, n_seq, begin, at, end);
                at = s.next;
                if (s.lo < s.hi) return true;
            }
            return false;
        }
        // item number n of all: its numbers are looked for by the sequences' items
        long long n = at < 0 ? blockIdx.x : at;
        at = n + gridDim.x;
        if (total == 0) return false;
        for (int i = 0; i < n_seq; ++i) {
            const int4 e = i < kAttEntries ? step[i] : *reinterpret_cast<const int4 *>(P.book + kKvHead + i * kKvStepWords);
            const long long items = e.z > 0 ? static_cast<long long>((e.z * g_heads + 127) / 128) * H : 0;
            if (n < items) {
                s = tree_segment(P, KT, prefix, step, n_seq, 0, prefix[i] * H + n * (tree_tiles(e.w, e.z, P.window, KT) + kTreeExtra), total);
                return true;
            }
            n -= items;
        }
        return false;
    };

    TreeSegment it;
    long long at = -1;
    if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptRegsLess));
    if (warp == 12) {
        int k = 0, v = 0, segments = 0;         // tiles of keys and of values that products have been issued for, segments
        int n_p[2] = {0, 0}, n_f[2] = {0, 0};
        auto score = [&](int x) {               // of key tile k
            att_wait(&k_full[k % ST], k / ST & 1, P.status);
            tc_fence_after();
            const uint32_t d = tm + x * 128, q0 = smem_u32(qs), k0 = smem_u32(ks + (k % ST) * A::kK);
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                tc_mma_f16(d, tc_smem_desc(q0 + i * 4096, 2048), tc_smem_desc(k0 + i * 2 * A::kKStep, A::kKStep), A::kIdescS, i > 0);
            if constexpr (SPLIT) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    tc_mma_f16(d, tc_smem_desc(q0 + A::kQ + i * 4096, 2048), tc_smem_desc(k0 + i * 2 * A::kKStep, A::kKStep), A::kIdescS, 1);
            }
            tc_commit_warp(&s_full[x]);
            tc_commit_warp(&k_free[k % ST]);
            if (lane == 0) mbar_arrive(&s_full[x]);         // what this thread saw of the keys' warps, for those who read the scales
            ++k;
        };
        // the scores' place is free: they have been read, or the weights that lie there have been used
        auto place_free = [&](int x) {
            if (n_p[x] == 0 && n_f[x] == 0) return;
            if (A::kApart) att_wait(&s_free[x], (n_f[x] - 1) & 1, P.status);
            else att_wait(&o_done[x], (n_p[x] - 1) & 1, P.status);
            tc_fence_after();
        };
        for (; next_segment(at, it); ++segments) {
            const int n = it.hi - it.lo;
            att_wait(&q_full, segments & 1, P.status);
            tc_fence_after();
            for (int j = 0; j < X && j < n; ++j) {
                place_free(j);
                score(j);
                ++n_f[j];
            }
            for (int j = 0; j < n; ++j, ++v) {
                const int x = X == 2 ? j & 1 : 0;
                if constexpr (A::kApart) {
                    if (j + X < n) {
                        place_free(x);
                        score(x);
                        ++n_f[x];
                    }
                }
                att_wait(&v_full[v % ST], v / ST & 1, P.status);
                att_wait(&p_full[x], n_p[x] & 1, P.status);
                tc_fence_after();
                const uint32_t d = tm + A::kColO + x * D, p = tm + (A::kApart ? A::kColP + x * A::kWidthP : x * 128), v0 = smem_u32(vs + (v % ST) * A::kV);
                const bool add = j / X % A::kChain != 0;
#pragma unroll
                for (int i = 0; i < KT / 16; ++i) {
                    const uint64_t desc = tc_smem_desc(v0 + i * 2 * A::kVStep, A::kVStep);
                    tc_mma_f16_t(d, p + i / 2 * kPartP + i % 2 * 8, desc, A::kIdescO, add || i > 0);
                    if constexpr (SPLIT) tc_mma_f16_t(d, p + i / 2 * kPartP + i % 2 * 8 + 16, desc, A::kIdescO, 1);
                }
                tc_commit_warp(&o_done[x]);
                tc_commit_warp(&v_free[v % ST]);
                ++n_p[x];
                if constexpr (!A::kApart) {
                    if (j + X < n) {
                        place_free(x);
                        score(x);
                        ++n_f[x];
                    }
                }
            }
        }
        for (int x = 0; x < X; ++x)
            if (n_p[x] > 0) tc_drain(&o_done[x], (n_p[x] - 1) & 1);
    } else if (warp >= 8 && warp < 12) {
        // A thread's codes of a tile are asked for a tile ahead, into places of its own (of segments too: what it does with them does not depend on where they come from).
        const int shift = P.s.page_shift, ct = tid - 256, cw = warp - 8, g = lane >> 2, t = lane & 3;
        constexpr int KU = KT * D / 16 / 128, KB = KU < 8 ? KU : 8;         // of 16 bytes: of a thread, at once
        constexpr int VU = SUBS * (D / 32) / 4, VB = VU < 8 ? VU : 8;          // of 512 bytes (16 tokens of 32 elements of a value): of a warp, at once
        const int k_row = ct % KT, k_sub = k_row >> 4, k_place = k_row & 15, k_token = (k_place >> 2) * 2 + (k_place & 1) + ((k_place & 2) << 2);
        uint4 *raw_k = reinterpret_cast<uint4 *>(raws) + ct, *raw_v = raw_k + KU * 128;
        // Pages and scales are looked up for 32 sub-blocks at a time, a lane each, and for the next 32 beside the work on these (behind the last sub-block: the last one).
        constexpr int GROUP = 32 / SUBS;        // tiles
        int tile = 0, group = 0, last_sub = 0;
        const int *table = nullptr;
        const uint8_t *head = nullptr;
        size_t from = 0, from_next = 0;
        float2 sc = make_float2(0.0f, 0.0f), sc_next = sc;
        float4 mine = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float zero = 0.0f;          // what stands for a scale of 0
        it.hi = 0;
        auto look_up = [&](int first_tile) {
            const int sub = min(first_tile * SUBS + lane, last_sub), page = table[sub >> (shift - 4)], in_page = sub & ((1 << (shift - 4)) - 1);
            from_next = static_cast<size_t>(page) * kv_page_bytes(P.s) + static_cast<size_t>(in_page) * (16 * D);
            if (cw == 0) sc_next = *reinterpret_cast<const float2 *>(P.scales + (static_cast<size_t>(page) * H + it.head) * 2);
        };
        auto take_over = [&]() {
            from = from_next, sc = sc_next;
            group = tile;
            if (group + GROUP < it.hi) look_up(group + GROUP);
            const float vsc = sc.y > 0.0f ? sc.y : zero, up = static_cast<float>(1 << kAttScale);
            if (cw == 0) mine = make_float4(sc.x, log2f(vsc), 1.0f / (up * vsc), up * sc.y);
        };
        auto next_tile = [&]() {
            if (++tile >= it.hi) {
                if (!next_segment(at, it)) return false;
                table = P.table + static_cast<size_t>(it.seq) * P.s.max_pages;
                last_sub = (it.length - 1) >> 4;
                head = P.pool + it.head * kv_head_bytes(P.s);
                if (cw == 0) zero = kv_zero_scale(P.reach[it.head]);
                tile = it.lo;
                look_up(tile);
                take_over();
            } else if (tile == group + GROUP) {
                take_over();
            }
            return true;
        };
        auto lane_of = [&](int sub) { return (tile - group) * SUBS + sub; };
        auto fetch = [](uint4 *to, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(src) : "memory"); };
        // keys: unit u is 16 elements of token u % KT; values: unit i * 4 + warp
        auto key_at = [&](const uint8_t *kp, int i) {
            const int k16 = (i * 128 + ct) / KT * 16;
            return reinterpret_cast<const uint4 *>(kp + k16 / CW * (16 * CW) + k16 % CW);
        };
        auto key_base = [&]() { return head + __shfl_sync(0xffffffffu, from, lane_of(k_sub)) + k_token * CW; };
        auto value_at = [&](int i) {
            const int u = i * 4 + cw, s = u / (D / 32), blk = u % (D / 32);
            return reinterpret_cast<const uint4 *>(head + __shfl_sync(0xffffffffu, from, lane_of(s)) + kv_half_bytes(P.s) + blk * 512 + lane * 16);
        };
        bool more = next_tile();
        auto ask_keys = [&]() {
            if (more) {
                const uint8_t *kp = key_base();
#pragma unroll
                for (int i = 0; i < KU; ++i) fetch(raw_k + i * 128, key_at(kp, i));
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto ask_values = [&]() {
            if (more) {
#pragma unroll
                for (int i = 0; i < VU; ++i) fetch(raw_v + i * 128, value_at(i));
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        ask_keys();
        ask_values();
        for (int n = 0; more; ++n) {
            const float4 of_tile = mine;
            const int scale_lane = lane - (tile - group) * SUBS, st = n % ST;
            const uint32_t par = (static_cast<uint32_t>(n / ST) & 1u) ^ 1u;
            uint4 u[KB], w[VB];
            more = next_tile();
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            att_wait(&k_free[st], par, P.status);
#pragma unroll
            for (int b = 0; b < KU; b += KB) {
#pragma unroll
                for (int i = 0; i < KB; ++i) u[i] = raw_k[(b + i) * 128];
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    const int k16 = ((b + i) * 128 + ct) / KT;
                    uint4 *to = reinterpret_cast<uint4 *>(ks + st * A::kK + k16 * 2 * A::kKStep + k_row * 16);
                    uint4 lo, hi;
                    kv_halves<E4M3>(u[i].x, lo.x, lo.y);
                    kv_halves<E4M3>(u[i].y, lo.z, lo.w);
                    kv_halves<E4M3>(u[i].z, hi.x, hi.y);
                    kv_halves<E4M3>(u[i].w, hi.z, hi.w);
                    to[0] = lo;
                    to[A::kKStep / 16] = hi;
                }
            }
            if (cw == 0 && scale_lane >= 0 && scale_lane < SUBS) scales[n & (A::kScales - 1)][scale_lane] = of_tile;
            fence_proxy_async();
            mbar_arrive(&k_full[st]);
            ask_keys();
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            att_wait(&v_free[st], par, P.status);
#pragma unroll
            for (int b = 0; b < VU; b += VB) {
#pragma unroll
                for (int i = 0; i < VB; ++i) w[i] = raw_v[(b + i) * 128];
#pragma unroll
                for (int i = 0; i < VB; ++i) {
                    const int unit = (b + i) * 4 + cw, s = unit / (D / 32), blk = unit % (D / 32);
                    uint8_t *to = vs + st * A::kV + (2 * s + (t >> 1)) * A::kVStep + (blk * 32 + g) * 16 + (t & 1) * 8;
                    const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint2 h;
                        kv_halves<E4M3>(words[j], h.x, h.y);
                        *reinterpret_cast<uint2 *>(to + j * 128) = h;
                    }
                }
            }
            fence_proxy_async();
            mbar_arrive(&v_full[st]);
            ask_values();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (warp < 4 * X) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptRegsMore));
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lanes = tm + (static_cast<uint32_t>((warp & 3) * 32) << 16), sc = lanes + x * 128, oc = lanes + A::kColO + x * D, pc = A::kApart ? lanes + A::kColP + x * A::kWidthP : sc;
        int n_s = 0, n_o = 0, n = 0;            // scores, sums, and tiles of all segments so far
        int cut_end = -1;                       // CTA in which the last item ends, where it is cut
        auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(128 * X) : "memory"); };
        for (int turn = 0; next_segment(at, it); ++turn) {
            const int row = it.item_row + r, last = it.rows - 1, start = it.length - it.count, node = min(row, last) / g_heads, tiles = it.hi - it.lo;         // (tiles of the segment)
            const bool is = row <= last;
            const int parent = r < it.count && x == 0 ? P.parents[it.row0 + r] : -1;        // (asked for in front of q, used behind it)
            // q: a warp brings eight rows at a time, a lane eight elements in front of every 32 of row lane % 8; the row's largest magnitude, then its F16 terms; element k
            // of row r lies at (k / 8) 2048 + r 16
            auto bring = [&](const auto *q) {
                using R = std::remove_const_t<std::remove_pointer_t<decltype(q)>>;
                constexpr int N = sizeof(R) / 2, U = D / 32, ROWS = 128 / (4 * X);         // 16 bytes of eight elements; eights of a lane; rows of a warp
#pragma unroll 2
                for (int r8 = warp * ROWS; r8 < (warp + 1) * ROWS; r8 += 8) {
                    const int q_row = r8 + (lane & 7), in = it.item_row + q_row;
                    const R *from = q + static_cast<size_t>(it.row0 + in / g_heads) * P.q_stride + (static_cast<size_t>(it.head) * g_heads + in % g_heads) * D + (lane >> 3) * 8;
                    uint4 u[U * N];
                    if (in >= it.rows) {
#pragma unroll
                        for (int i = 0; i < U * N; ++i) u[i] = make_uint4(0, 0, 0, 0);
                    } else if (P.vec) {
#pragma unroll
                        for (int i = 0; i < U * N; ++i) u[i] = *reinterpret_cast<const uint4 *>(from + i / N * 32 + i % N * (8 / N));
                    } else {
#pragma unroll
                        for (int i = 0; i < U; ++i) {
                            __align__(16) R y[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) y[j] = from[i * 32 + j];
#pragma unroll
                            for (int j = 0; j < N; ++j) u[i * N + j] = reinterpret_cast<const uint4 *>(y)[j];
                        }
                    }
                    auto number = [&](int i) { return static_cast<float>(reinterpret_cast<const R *>(&u[i / (8 / N)])[i % (8 / N)]); };
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8 * U; ++i) top = fmaxf(top, fabsf(number(i)));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const int e = top > 0.0f ? max(-100, min(128, static_cast<int>(__float_as_uint(top) >> 23) - 126)) - 15 : 0, e1 = e / 2, e2 = e - e1;
                    if (lane < 8) muls[q_row] = P.scale_log2 * __uint_as_float((127 + e1) << 23) * __uint_as_float((127 + e2) << 23);
                    const float down = __uint_as_float((127 - e1) << 23), down2 = __uint_as_float((127 - e2) << 23);
                    uint8_t *to = qs + (lane >> 3) * 2048 + q_row * 16;
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float a = number(8 * i + 2 * j) * down * down2, b = number(8 * i + 2 * j + 1) * down * down2;
                            hi[j] = half_pair(a, b);
                            if constexpr (SPLIT) lo[j] = half_rest(a, b, hi[j]);
                        }
                        *reinterpret_cast<uint4 *>(to + i * 4 * 2048) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        if constexpr (SPLIT) *reinterpret_cast<uint4 *>(to + A::kQ + i * 4 * 2048) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            };
            if constexpr (SPLIT) bring(static_cast<const float *>(P.q));
            else if (P.type == kRowsF16) bring(static_cast<const __half *>(P.q));
            else bring(static_cast<const __nv_bfloat16 *>(P.q));
            if (r < it.count && x == 0) places[turn & 1][r] = static_cast<int8_t>(parent >= 0 && parent < r ? parent : -1);
            fence_proxy_async();
            mbar_arrive(&q_full);
            meet();             // (the parents and the factors are there)
            const float mul = muls[r];
            float m = kAttFloor, l = 0.0f;
            int mine = 0;       // this stream's tiles so far
            // the row's maximum is now `most` or what it was; brought to it where it has grown enough
            auto follow = [&](float most) {
                if (mine == 0) {
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
            auto work = [&](auto apart) {
                constexpr bool kFar = decltype(apart)::value;
#pragma unroll 1
                for (int j = x; j < tiles;) {
                    const int chain_end = min(j + A::kChain * X, tiles);
#pragma unroll 1
                    for (; j < chain_end; j += X, ++mine) {
                        const int first = (it.lo + j) * KT;
                        const float4 *scale = scales[(n + j) & (A::kScales - 1)];
                        att_wait(&s_full[x], n_s++ & 1, P.status);
                        tc_fence_after();
                        const bool edge = first + KT - 1 >= start || (P.window && first <= start + it.count - 1 - P.window);
                        TreeSight sight = {~0ull, ~0ull};
                        if (edge) sight = tree_sight(places[turn & 1], node, start, first, P.window);
                        // column 16 s + p of the scores is token 2 (p / 4) + (p & 1) + 8 ((p & 3) / 2) of sub-block s
                        auto hidden = [&](int c, int i) {
                            const int p = i & 15, in = (i & 16) + (p >> 2) * 2 + (p & 1) + ((p & 2) << 2);
                            return !((c & 2 ? sight.hi : sight.lo) >> ((c & 1) * 32 + in) & 1ull);
                        };
                        if constexpr (kFar) {           // (rare: little code, few registers, the scores read twice)
                            float most = kAttFloor;
                            uint32_t u[32], hi[16], lo[16];
                            auto scores = [&](int c) {          // of the 32 tokens from 32 c on
                                tc_ld(sc + c * 32, u);
                                tc_wait_ld(u);
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (hidden(c, i)) u[i] = 0xff800000u;
                            };
#pragma unroll 1
                            for (int c = 0; c < KT / 32; ++c) {
                                scores(c);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float4 s4 = scale[2 * c + i / 16];
                                    most = fmaxf(most, fmaf(__uint_as_float(u[i]), fmaxf(mul * s4.x, 1e-37f), s4.y));
                                }
                            }
                            if constexpr (A::kApart) {
                                if (n_o > 0) att_wait(&o_done[x], (n_o - 1) & 1, P.status);
                                tc_fence_after();
                            }
                            follow(most);
                            const float off = (A::kTop - static_cast<float>(kAttScale)) - m;
#pragma unroll 1
                            for (int c = 0; c < KT / 32; ++c) {
                                scores(c);
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const float4 s4 = scale[2 * c + i / 8];
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
                            if (edge) {
#pragma unroll
                                for (int c = 0; c < KT / 32; ++c)
#pragma unroll
                                    for (int i = 0; i < 32; ++i)
                                        if (hidden(c, i)) v[c][i] = 0xff800000u;
                            }
                            float most = kAttFloor;
#pragma unroll
                            for (int b = 0; b < SUBS; ++b) {
                                const float4 s4 = scale[b];
                                auto of = [&](int i) { return __uint_as_float(v[b / 2][b % 2 * 16 + i]); };
                                float t = max3(of(0), of(1), of(2));
#pragma unroll
                                for (int i = 3; i < 15; i += 2) t = max3(t, of(i), of(i + 1));
                                t = fmaxf(t, of(15));
                                most = fmaxf(most, fmaf(t, fmaxf(mul * s4.x, 1e-37f), s4.y));
                            }
                            if constexpr (A::kApart) {          // the sums, and the place of the weights, are free
                                if (n_o > 0) att_wait(&o_done[x], (n_o - 1) & 1, P.status);
                                tc_fence_after();
                            }
                            follow(most);
                            const float base = m - A::kTop;
                            // exponents of all columns, then the exponentials (scales read between the stores of weights would wait for them)
#pragma unroll
                            for (int b = 0; b < SUBS; ++b) {
                                const float4 s4 = scale[b];
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
                                l = fmaf(a + c, scale[b].z, l);
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
                    if (j < tiles) {
                        int of = r;
                        asm volatile("" : "+r"(of));          // (addresses are made here, not held through the tiles)
                        const int place = blockIdx.x * kTreeUnits + 1 + x;
                        const bool more = mine > A::kChain;
                        float *held_m = &prompt_part_end<D, 128>(P.part, place, of)->x;
                        const float f = more ? ex2(*held_m - m) : 0.0f;         // (m does not go down)
                        *held_m = m;
                        float4 h[8];
                        auto ask = [&](int c) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) h[i] = more ? *reinterpret_cast<const float4 *>(prompt_part<D, 128>(P.part, place, of, c + 4 * i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
                            for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(prompt_part<D, 128>(P.part, place, of, c + 4 * i)) = y[i];
                        }
                        tc_fence_before();
                    }
                }
            };
            if (kv_far_apart(P.reach[it.head])) work(std::true_type{});
            else work(std::false_type{});
            n += tiles;
            // ---- the segment's end: each stream's maximum, denominator, and what brings the sums of the chains in front of its last one to its maximum
            if (mine > 0) att_wait(&o_done[x], (n_o - 1) & 1, P.status);
            int of = r;
            asm volatile("" : "+r"(of));
            const int unit = blockIdx.x * kTreeUnits;
            ends[x][r] = make_float4(m, l, mine > A::kChain ? ex2(prompt_part_end<D, 128>(P.part, unit + 1 + x, of)->x - m) : 0.0f, mine > A::kChain ? 1.0f : 0.0f);
            meet();
            tc_fence_after();
            float4 en[X];
            float all = kAttFloor, den = 0.0f, f[X];
#pragma unroll
            for (int i = 0; i < X; ++i) en[i] = ends[i][r], all = fmaxf(all, en[i].x);
#pragma unroll
            for (int i = 0; i < X; ++i) {
                const float half_way = ex2(0.5f * (en[i].x - all));
                f[i] = half_way * half_way;
                den += en[i].y * half_way * half_way;
            }
            // 16 columns of the sums
            auto sums = [&](int c, float (&y)[16]) {
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = 0.0f;
#pragma unroll
                for (int w = 0; w < X; ++w) {
                    if (w >= tiles) continue;           // (a stream without a tile has no sums)
                    uint32_t v[16];
                    tc_ld(lanes + A::kColO + w * D + c * 16, v);
                    tc_wait_ld(v);
                    if (en[w].w != 0.0f) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 h = *reinterpret_cast<const float4 *>(prompt_part<D, 128>(P.part, unit + 1 + w, of, c * 16 + i));
                            v[i] = __float_as_uint(fmaf(h.x, en[w].z, __uint_as_float(v[i])));
                            v[i + 1] = __float_as_uint(fmaf(h.y, en[w].z, __uint_as_float(v[i + 1])));
                            v[i + 2] = __float_as_uint(fmaf(h.z, en[w].z, __uint_as_float(v[i + 2])));
                            v[i + 3] = __float_as_uint(fmaf(h.w, en[w].z, __uint_as_float(v[i + 3])));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = fmaf(__uint_as_float(v[i]), f[w], y[i]);
                }
            };
            const float inv = kAttUnit / den;
            const int to_unit = unit + (it.begun ? 0 : 1);
            const size_t dst = static_cast<size_t>(it.row0 + row / g_heads) * P.out_stride + (static_cast<size_t>(it.head) * g_heads + row % g_heads) * D;
            // 16 elements of the row's answer from c on
            auto answer = [&](int c, const float (&y)[16]) {
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
                if constexpr (SPLIT) put(static_cast<float *>(P.out) + dst + c);
                else if (P.type == kRowsF16) put(static_cast<__half *>(P.out) + dst + c);
                else put(static_cast<__nv_bfloat16 *>(P.out) + dst + c);
            };
#pragma unroll 1
            for (int c = x * (D / X); c < (x + 1) * (D / X); c += 16) {
                float y[16];
                sums(c / 16, y);
                if (is && !it.whole) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) __stcg(reinterpret_cast<float4 *>(prompt_part<D, 128>(P.part, to_unit, of, c + i)), make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]));
                } else if (is) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] *= inv;
                    answer(c, y);
                }
                __syncwarp();
            }
            if (is && !it.whole && x == 0) *prompt_part_end<D, 128>(P.part, to_unit, of) = make_float2(all, den);
            if (tid == 0 && P.split && !it.begun && it.tile1 > end) {
                P.cuts[2 * blockIdx.x] = make_int4(it.row0, it.rows, it.head, it.item_row);
                cut_end = static_cast<int>((it.tile1 - 1) / chunk);
            }
            tc_fence_before();      // the sums have been read: the next segment's may be written once its weights are there
            meet();
        }
        if (P.split && tid == 0) P.cuts[2 * blockIdx.x + 1] = make_int4(cut_end, 0, 0, 0);
    } else if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptRegsMore));
    }
    grid_dep_launch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
}

// The parts of the items that several CTAs have one of: blockIdx.x is the CTA that an item begins in, blockIdx.y some of its rows; a thread has four elements of a row.
template <int D>
constexpr int kTreeJoinRows = D == 96 ? 8 : 1024 / D;
template <int D>
__global__ void __launch_bounds__(256) kv_tree_join_kernel(const __grid_constant__ KvTree P) {
    grid_dep_wait();
    const int c0 = blockIdx.x, tid = threadIdx.x, r = blockIdx.y * kTreeJoinRows<D> + tid / (D / 4), c = tid % (D / 4) * 4;
    const int4 a = P.cuts[2 * c0], b = P.cuts[2 * c0 + 1];
    if (b.x < 0 || tid / (D / 4) >= kTreeJoinRows<D> || a.w + r >= a.y) return;
    const int g_heads = P.s.heads / P.s.kv_heads, row = a.w + r;
    float top = kAttFloor, den = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int k0 = c0; k0 <= b.x; k0 += 8) {
        float2 z[8];
        float4 y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int from = min(k0 + k, b.x), unit = from * kTreeUnits + (from == c0 ? 1 : 0);       // (of the others it is the first item)
            z[k] = *prompt_part_end<D, 128>(P.part, unit, r);
            y[k] = *reinterpret_cast<const float4 *>(prompt_part<D, 128>(P.part, unit, r, c));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k0 + k > b.x) break;
            const float both = fmaxf(top, z[k].x), ha = ex2(0.5f * (top - both)), hb = ex2(0.5f * (z[k].x - both)), fa = ha * ha, fb = hb * hb;
            top = both;
            den = den * ha * ha + z[k].y * hb * hb;
            sum.x = fmaf(y[k].x, fb, sum.x * fa), sum.y = fmaf(y[k].y, fb, sum.y * fa), sum.z = fmaf(y[k].z, fb, sum.z * fa), sum.w = fmaf(y[k].w, fb, sum.w * fa);
        }
    }
    const float inv = kAttUnit / den;
    const size_t to = static_cast<size_t>(a.x + row / g_heads) * P.out_stride + (static_cast<size_t>(a.z) * g_heads + row % g_heads) * D + c;
    auto put = [&](auto *o) {
        using R = std::remove_pointer_t<decltype(o)>;
        __align__(16) R v[4] = {row_number<R>(sum.x * inv), row_number<R>(sum.y * inv), row_number<R>(sum.z * inv), row_number<R>(sum.w * inv)};
        if (P.vec) {
            if constexpr (sizeof(R) == 4) *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(v);
            else *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = v[i];
        }
    };
    if (P.type == kRowsF32) put(static_cast<float *>(P.out) + to);
    else if (P.type == kRowsF16) put(static_cast<__half *>(P.out) + to);
    else put(static_cast<__nv_bfloat16 *>(P.out) + to);
}

}  // namespace wd
