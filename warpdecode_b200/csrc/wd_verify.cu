// Verification of drafted tokens against the target's probabilities, from given random numbers (wd_verify_drafts).
//
// p = softmax(x / T), q the draft's. At a row whose children were drawn from q, what is left of p after j rejections is proportional to max(p - c_j q, 0):
//   c_0 = 0,  S(c) = sum max(p - c q, 0),  c_(j + 1) = c_j + S(c_j)
// (one rejection makes max(r - q, 0) / Z of r = max(p - c q, 0) / S, and max(max(p - c q, 0) / S - q, 0) S = max(p - (c + S) q, 0)), so that nothing of the
// vocabulary's size is kept from one child to the next, and a number each decides: u S q(x) < max(p(x) - c q(x), 0).
//
// A cluster of CTAs goes down a sequence's tree and reads the rows on its way alone, not those of all drafts. A row's maximum and sum are F32 and decide
// for a child that is not within 1e-4 of its border, or more where a thread has very many terms. What is nearer, and every draw, is made of sums in 64 bits: the running sums
// of 150,000 tokens lie 1e-7 apart where the unlikely ones are, and the heavy ones' F32 errors (3e-8) would choose among them.
//
// A warp has a run of the vocabulary, the warps of a cluster one behind the other. It copies its part of a row into shared memory, where all of the row's passes
// read it, and where there are few sequences that of the rows that may be next beside it. What a CTA finds it sends to all CTAs' shared memory, where 16 bytes from
// each complete a barrier (550 cycles; behind a barrier of the cluster it is 1,000), and every warp puts them together by the same arithmetic and comes to the same
// decision, so that nothing is sent back.
//
// 64 chains of 5 rows of 151,936 F32, with a draft: 137 to 141 us (33 at the memory's rate; DRAM 18 % busy, 1.9 instructions a cycle, the pipe of 64 bits 11 %). 14 clusters of 16 CTAs
// run at once, and there each holds one row: a CTA waits for its part of the row, then works on it with nothing on its way, 32 us for each further accepted row (16 without a
// draft). One chain 21 to 32, 3 to 3.5 a row and 7 a draw, bound by latency. With rows read from memory by each pass, sums met by a barrier of the cluster, and exp() for the
// terms 250 and 41.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <type_traits>

#include "wd_device.cuh"
#include "wd_host.h"

namespace cg = cooperative_groups;
using wd_host::OnDevice;
using wd_host::set_error;

namespace wd {
namespace {

constexpr int kVerThreads = 256, kVerWarps = kVerThreads / 32, kVerCtas = 16, kVerRows = 1024, kVerSlots = 4;
constexpr float kVerGreedy = 1e-6f, kVerFloor = -3.402823466e38f;
// How near its border, relative to the numbers that are compared, a child is left to the sums in 64 bits. Exponents are off by three roundings of up to 120 (2^-16 of a term),
// a lane's sum of n terms by 11 roundings of 2^-24 for every ten: four of the exponential by which it follows a larger maximum, one of that product, six of additions.
// Together less than 3e-5 and n 2^-23 of a probability. 1e-4 is more than that up to 580 terms a lane: 2.3 million tokens by 16 CTAs, 148,000 by one.
constexpr float kVerUnsure = 1e-4f;
inline float ver_unsure(int piece) { return fmaxf(kVerUnsure, 3e-5f + 0x1p-23f * static_cast<float>(piece)); }

struct VerifyParams {
    const void *target, *draft;
    long long target_stride, draft_stride;
    int rows, vocab, n_seqs, ctas, slots, run_bytes, piece;         // slots: rows that shared memory holds of target and draft; run_bytes: of a warp's run in it, 0: it holds none; piece: of a lane
    const int *first, *tokens, *parents;
    const float *uniforms, *temperature;
    int *path, *count, *next;
    float unsure;           // see ver_unsure
    int stop_at, stop_rank, stop_warp;      // tests: the meeting whose wait runs out, -1: none; in which CTA, in which of its warps, -1: in all
    double power[32];       // 2^(j / 32)
};

__device__ __forceinline__ float ver_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float ver_max(float a, float b) {        // a NaN stays one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

struct RowSum {             // s = sum 2^(k (x - m)); m is a NaN or +inf where the row has no distribution
    float m, s;
};
// larger numbers above (of a NaN nothing is said)
__device__ __forceinline__ uint32_t ver_order(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float ver_warp_max(float x) {        // a NaN stays one
    const uint32_t o = __reduce_max_sync(0xffffffffu, ver_order(x));
    return __any_sync(0xffffffffu, x != x) ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
template <class N>
__device__ __forceinline__ N ver_warp_sum(N x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// 2^(k32 d / 32), d <= 0, for k32 d > -32,000: by a table of 2^(j / 32) and the series of the rest (Tang, ACM TOMS 15, 1989), off by 2^-48. Half the work of exp().
__device__ __forceinline__ double ver_power(const double *table, double d, double k32) {
    constexpr double ln = 0.693147180559945309417232 / 32, magic = 6755399441055744.0;       // 1.5 2^52: what is added to it is rounded to a whole number
    const double y = fma(d, k32, magic), r = fma(d, k32, magic - y);
    const int n = __double2loint(y);
    double v = fma(r, ln * ln * ln * ln * ln / 120, ln * ln * ln * ln / 24);
    v = fma(r, v, ln * ln * ln / 6);
    v = fma(r, v, ln * ln / 2);
    v = fma(r, v, ln);
    v = fma(r, v, 1.0) * table[n & 31];
    return __hiloint2double(__double2hiint(v) + (n >> 5) * (1 << 20), __double2loint(v));
}

struct VerifyShared {
    uint4 slot[2][kVerCtas][3], warp_slot[2][kVerWarps][3];     // what the CTAs of a cluster, and the CTA's warps, bring, in turn
    uint64_t full[2];
    double power[32], lane_sum[kVerWarps][32], lane_bend[kVerWarps][32];
    int rejected[kVerRows];                             // tokens
    int gone_at;                                        // the barrier that a warp came to after a wait that ran out
    int16_t parents[kVerRows], kids[kVerWarps][32], path[kVerRows];
};
struct VerOne {
    uint4 v[1];
};
struct VerThree {
    uint4 v[3];
};
// to the same place of another CTA of the cluster, and to its barrier
__device__ __forceinline__ void ver_send(uint4 *to, uint64_t *bar, int cta, uint4 v) {
    asm volatile(
        "{\n .reg .b32 a, b;\n mapa.shared::cluster.u32 a, %0, %2;\n mapa.shared::cluster.u32 b, %1, %2;\n"
        " st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [a], {%3, %4, %5, %6}, [b];\n}" ::"r"(smem_u32(to)),
        "r"(smem_u32(bar)), "r"(cta), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
        : "memory");
}

// whether the barrier's phase was completed within a second
__device__ __forceinline__ bool ver_wait(uint64_t *bar, uint32_t parity) {
    unsigned long long t0 = 0;
#pragma unroll 1
    for (unsigned i = 1; !mbar_try_wait(bar, parity); ++i) {
        if (i % 64 != 0) continue;          // (the timer is slow to read, and an ordinary wait is over before)
        const unsigned long long t = global_timer_ns();
        if (i == 64) t0 = t;
        else if (t - t0 > kWaitLimitNs) return false;
    }
    return true;
}

enum { kSumFirst, kSumLeft, kSumTarget };   // of p, of q and of max(p - q, 0); of max(p - c q, 0); of p without the rejected tokens

// Among a warp's K numbers a lane (in order: lane, then place), `base` in front of them: the first one whose running sum is above the aim, else the last one that is
// not 0. Returns its place, -1 where all are 0; base becomes what is in front of it.
template <int K>
__device__ __forceinline__ int ver_pick(const double (&v)[K], double aim, double &base, int lane) {
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < K; ++i) own += v[i];
    double upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    double at = __shfl_up_sync(0xffffffffu, upto, 1);
    at = base + (lane ? at : 0.0);
    int place = -1;
    bool above = false;
    double front = at;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        if (v[i] > 0.0 && !above) place = i, front = at, above = at + v[i] > aim;
        at += v[i];
    }
    const unsigned first = __ballot_sync(0xffffffffu, above), some = __ballot_sync(0xffffffffu, place >= 0);
    const int from = first ? __ffs(first) - 1 : 31 - __clz(some);
    if (!some) return -1;
    base = __shfl_sync(0xffffffffu, front, from);
    return from * K + __shfl_sync(0xffffffffu, place, from);
}

// (registers for three CTAs an SM where there is no draft; with one, shared memory has room for two at most, and they may have them)
template <class T, bool HELD, bool DRAFT>
__global__ void __launch_bounds__(kVerThreads, DRAFT ? 2 : 3) verify_kernel(const __grid_constant__ VerifyParams P) {
    extern __shared__ __align__(16) uint8_t ver_rows[];
    __shared__ VerifyShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = P.ctas, rank = ctas > 1 ? static_cast<int>(cluster.block_rank()) : 0, seq = static_cast<int>(blockIdx.x) / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = P.vocab, me = rank * kVerWarps + warp;
    const int share = P.rows / P.n_seqs;
    const int f0 = P.first ? min(max(P.first[seq], 0), P.rows) : seq * share, f1 = P.first ? min(max(P.first[seq + 1], f0), P.rows) : f0 + share, n = f1 - f0;
    if (n == 0 || n > kVerRows) {
        if (rank == 0) {
            for (int i = tid; i < n; i += kVerThreads) P.path[f0 + i] = -1;
            if (tid == 0) P.count[seq] = 0, P.next[seq] = -1;
        }
        return;
    }
    if (ctas > 1) {
        if (tid == 0) {
            mbar_init(&sh.full[0], 1);
            mbar_init(&sh.full[1], 1);
            mbar_fence_init();
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");         // (waited for before anything is sent)
    }
    const float heat = P.temperature ? P.temperature[seq] : 1.0f;
    constexpr float none = -INFINITY;
    // A warp's run is 32 pieces of `piece` elements, a lane's each, one behind the other: so the lanes' sums are sums of what lies together, and the search for a
    // token ends in one piece. (An odd number: the lanes read from different banks.)
    const int piece = P.piece;
    auto run_begin = [&](int run) { return static_cast<int>(min(static_cast<long long>(run) * piece * 32, static_cast<long long>(vocab))); };
    const int run0 = run_begin(me), mine_n = run_begin(me + 1) - run0, lane0 = min(lane * piece, mine_n), lane1 = min(lane0 + piece, mine_n);
    auto target_row = [&](int i) { return static_cast<const T *>(P.target) + static_cast<size_t>(f0 + i) * P.target_stride; };
    auto draft_row = [&](int i) { return static_cast<const T *>(P.draft) + static_cast<size_t>(f0 + i) * P.draft_stride; };

    // ---- rows in shared memory: a slot is [target, draft][warps] of run_bytes; a run lies in it as in memory, from the boundary of 16 bytes in front of it on
    auto run_place = [&](int slot, int which, int w) { return ver_rows + (static_cast<size_t>(slot) * (DRAFT ? 2 : 1) + which) * kVerWarps * P.run_bytes + static_cast<size_t>(w) * P.run_bytes; };
    auto beside = [](const T *x) { return static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15u); };
    auto copy_run = [&](const T *x, uint8_t *to) {
        const T *from = x + run0;
        const int off = beside(from), lead = min(off ? (16 - off) / static_cast<int>(sizeof(T)) : 0, mine_n), chunks = (mine_n - lead) * static_cast<int>(sizeof(T)) / 16;
        const int tail = lead + chunks * 16 / static_cast<int>(sizeof(T)), loose = lead + mine_n - tail;
        const uint32_t dst = smem_u32(to + off + lead * sizeof(T));
        for (int i = lane; i < chunks; i += 32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * 16), "l"(reinterpret_cast<const uint8_t *>(from + lead) + i * 16) : "memory");
        if (lane < loose) {                 // single elements in front of the first boundary and behind the last
            const int i = lane < lead ? lane : tail + lane - lead;
            reinterpret_cast<T *>(to + off)[i] = from[i];
        }
    };
    int slot_node[kVerSlots], issued = 0;
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < kVerSlots; ++i) slot_node[i] = -1;
    }
    auto ask = [&](int node, bool draft) {
        __syncwarp();                       // (what was there has been read)
        const int slot = issued % P.slots;
        copy_run(target_row(node), run_place(slot, 0, warp));
        if (draft) copy_run(draft_row(node), run_place(slot, 1, warp));
        asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
        for (int i = 0; i < kVerSlots; ++i)
            if (i == slot) slot_node[i] = node;
        ++issued;
    };

    if constexpr (HELD) copy_run(target_row(0), run_place(0, 0, warp));
    for (int i = tid; i < n; i += kVerThreads) {
        const int p = P.parents ? P.parents[f0 + i] : i - 1;
        sh.parents[i] = static_cast<int16_t>(p >= 0 && p < i ? p : -1);
    }
    if (tid < 32) sh.power[tid] = P.power[tid];
    if (tid == 0) sh.gone_at = 0x7fffffff;
    const bool greedy = !(heat >= kVerGreedy), with_draft = DRAFT && !greedy;
    const float k = greedy ? 1.44269504f : fmaxf(static_cast<float>(1.4426950408889634 / heat), 1e-30f);        // (not 0: -inf times k has to stay what it is)
    const double k32 = greedy ? 0.0 : 32 * 1.4426950408889634 / heat;
    if constexpr (HELD) {
        if (with_draft && n > 1) copy_run(draft_row(0), run_place(0, 1, warp));
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot_node[0] = 0;
        issued = 1;
    }
    __syncthreads();
    // What the warps of the cluster bring, put together by `join` (of a lane's 16 bytes, whether it has any; the same in all lanes). The places of a turn are free
    // again when all have come to the next one.
    int turn = 0, meetings = 0;
    // A wait that runs out in a warp (gone) is known to all of the CTA from that warp's next barrier on, whichever it is to the others (lost): the warp says which number it
    // has before it comes there. (__syncthreads_or() takes 150 ns more than a barrier.) From then on nothing is sent or waited for. What such a warp finds is zeros.
    bool gone = false, lost = false;
    int barriers = 0;
    const int stop_at = (P.stop_rank < 0 || rank == P.stop_rank) && (P.stop_warp < 0 || warp == P.stop_warp) ? P.stop_at : -1;
    auto all_here = [&]() __attribute__((always_inline)) {
        if (lost) return;
        ++barriers;
        if (gone) sh.gone_at = barriers;
        __syncthreads();
        lost = *static_cast<volatile int *>(&sh.gone_at) <= barriers;
    };
    auto meet = [&](auto mine, auto join) __attribute__((always_inline)) {          // (one or three times 16 bytes)
        constexpr int N = sizeof(mine) / 16;
        const decltype(mine) nothing{};
        if (lost) return nothing;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) sh.warp_slot[turn][warp][i] = mine.v[i];
        if (ctas > 1 && tid == 0) mbar_expect_tx(&sh.full[turn], 16 * N * ctas);
        all_here();
        auto all = mine;
        if (ctas == 1 || warp == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) all.v[i] = sh.warp_slot[turn][lane & (kVerWarps - 1)][i];
            all = join(all, lane < kVerWarps);
        }
        if (lost) return nothing;           // (asked behind the reading of the slots, which takes as long)
        if (ctas > 1) {
            if (meetings == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // (all have made their barriers)
            if (warp == 0 && lane < ctas)
#pragma unroll
                for (int i = 0; i < N; ++i) ver_send(&sh.slot[turn][rank][i], &sh.full[turn], lane, all.v[i]);
            gone = !__all_sync(0xffffffffu, meetings != stop_at && ver_wait(&sh.full[turn], meetings >> 1 & 1));
#pragma unroll
            for (int i = 0; i < N; ++i) all.v[i] = sh.slot[turn][lane & (kVerCtas - 1)][i];
            all = join(all, lane < ctas);
            if (gone) all = nothing;
        }
        turn ^= 1;
        ++meetings;
        return all;
    };

    const T *tp = nullptr, *dp = nullptr;   // the row's logits; of the draft: null where it is not asked
    int slot = 0;                           // where the row is held
    // where a run of the row is, warp w's, which begins at `begin`
    auto run_of = [&](int which, int w, int begin) {
        const T *x = (which ? dp : tp) + begin;
        if constexpr (HELD) return reinterpret_cast<const T *>(run_place(slot, which, w) + beside(x));
        else return x;
    };
    // maxima and sums of the row, and its largest logit
    RowSum sp{}, sq{};
    int best = 0;
    auto row_sums = [&]() __attribute__((always_inline)) {
        constexpr int U = 10;
        float m[2] = {kVerFloor, kVerFloor}, s[2] = {0.0f, 0.0f}, top = none;
        int top_at = 0;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (w == 1 && !dp) break;
            const T *x = run_of(w, warp, run0);
#pragma unroll 1
            for (int i = lane0; i < lane1; i += U) {
                float v[U];
#pragma unroll
                for (int j = 0; j < U; ++j) v[j] = i + j < lane1 ? static_cast<float>(x[i + j]) : none;
                float now = m[w], other = v[1];
#pragma unroll
                for (int j = 0; j < U; j += 2) now = ver_max(now, v[j]), other = ver_max(other, v[j + 1]);
                now = ver_max(now, other);
                if (greedy) {
#pragma unroll
                    for (int j = 0; j < U; ++j)
                        if (v[j] > top) top = v[j], top_at = run0 + i + j;          // (upwards: of equals the first one stays)
                } else {
                    float sum = s[w] * ver_ex2((m[w] - now) * k), more = 0.0f;
#pragma unroll
                    for (int j = 0; j < U; j += 2) {
                        sum += ver_ex2((v[j] - now) * k);
                        more += ver_ex2((v[j + 1] - now) * k);
                    }
                    s[w] = sum + more;
                }
                m[w] = now;
            }
        }
        if (greedy) {                       // the maximum, for what is no number; the largest logit, its place
            auto join = [&](const VerOne &x, bool is) {
                const uint4 v = x.v[0];
                const uint32_t o = is ? ver_order(__uint_as_float(v.y)) : 0u, most = __reduce_max_sync(0xffffffffu, o);
                const float any = ver_warp_max(is ? __uint_as_float(v.x) : kVerFloor);
                return VerOne{{make_uint4(__float_as_uint(any), most & 0x80000000u ? most & 0x7fffffffu : ~most, __reduce_min_sync(0xffffffffu, is && o == most ? v.z : 0x7fffffffu), 0u)}};
            };
            const uint4 all = meet(join(VerOne{{make_uint4(__float_as_uint(m[0]), __float_as_uint(top), static_cast<uint32_t>(top_at), 0u)}}, true), join).v[0];
            sp = RowSum{__uint_as_float(all.x), __uint_as_float(all.y)};
            best = static_cast<int>(all.z);
            return;
        }
        auto join = [&](const VerOne &x, bool is) {
            const uint4 v = x.v[0];
            const float pm = is ? __uint_as_float(v.x) : kVerFloor, qm = is ? __uint_as_float(v.z) : kVerFloor, p = ver_warp_max(pm);
            uint4 r = make_uint4(__float_as_uint(p), 0u, 0u, 0u);
            float ps = is ? __uint_as_float(v.y) * ver_ex2((pm - p) * k) : 0.0f;
            if (dp) {
                const float q = ver_warp_max(qm);
                r.z = __float_as_uint(q);
                r.w = __float_as_uint(ver_warp_sum(is ? __uint_as_float(v.w) * ver_ex2((qm - q) * k) : 0.0f));
            }
            r.y = __float_as_uint(ver_warp_sum(ps));
            return VerOne{{r}};
        };
        const uint4 all = meet(join(VerOne{{make_uint4(__float_as_uint(m[0]), __float_as_uint(s[0]), __float_as_uint(m[1]), __float_as_uint(s[1]))}}, true), join).v[0];
        sp = RowSum{__uint_as_float(all.x), __uint_as_float(all.y)};
        sq = RowSum{__uint_as_float(all.z), __uint_as_float(all.w)};
    };

    // ---- in 64 bits
    double over_zp = 0.0, over_zq = 0.0, c = 0.0, ratio = 0.0, bend = 0.0;
    int n_rejected = 0;
    auto power = [&](float v, float m) {
        // (0 where there is no term, or one below 2^-1000; -inf times a scale of 0 is a NaN; without a branch, so that several are made side by side)
        const bool is = (v - m) * k > -1000.0f;
        const double r = ver_power(sh.power, static_cast<double>(is ? v : m) - static_cast<double>(m), k32);
        return is ? r : 0.0;
    };
    auto is_rejected = [&](int x) {
        bool is = false;
#pragma unroll 1
        for (int j = 0; j < n_rejected; ++j) is |= sh.rejected[j] == x;
        return is;
    };
    // What is left of the target: max(p - c q, 0) zp = max(w - ratio v, 0) of the terms w and v of p and q, ratio = c zp / zq. So one pass finds zp, zq and what the
    // first rejection leaves, although it needs them: it takes the ratio that the F32 sums give, and beside the sum of the terms v that have something left. By the right
    // ratio the sum is less by the difference times that of v, but for terms that something is left of by one ratio and nothing by the other. Where the ratios are within
    // 2^-19 of each other, such a term's w - ratio v is below 2^-19 ratio v, and that below 2^-18 w: those terms' v are summed too. Where they could be felt (a draft that
    // is the target but for a few tokens), or the ratios are farther apart, a pass is made with the right one.
    auto left_of = [&](const T *x, const T *y, int i, double r) { return fmax(fma(-r, power(static_cast<float>(y[i]), sq.m), power(static_cast<float>(x[i]), sp.m)), 0.0); };
    // The whole cluster's sums (first: p, q and what is left of p; else one), the CTAs' of what a draw is made from in the slots, the warps' and the lanes' in their places.
    auto sums = [&](auto kind, double *found) __attribute__((always_inline)) {
        constexpr int KIND = decltype(kind)::value, U = KIND == kSumTarget ? 8 : 4;
        double a = 0.0, b = 0.0, d = 0.0, e = 0.0, near = 0.0;
        const T *x = run_of(0, warp, run0), *y = KIND == kSumTarget ? nullptr : run_of(1, warp, run0);
        auto add = [&](int i) {
            if (KIND == kSumTarget) {
                const double v = power(static_cast<float>(x[i]), sp.m);
                return n_rejected > 0 && is_rejected(run0 + i) ? 0.0 : v;
            }
            if (KIND == kSumLeft) return left_of(x, y, i, ratio);
            const double w = power(static_cast<float>(x[i]), sp.m), v = power(static_cast<float>(y[i]), sq.m), rest = fma(-ratio, v, w);
            b += w;
            d += v;
            e += rest > 0.0 ? v : 0.0;
            near += (__double2hiint(rest) & 0x7fffffff) + (18 << 20) < __double2hiint(w) ? v : 0.0;
            return fmax(rest, 0.0);
        };
        int i = lane0;
#pragma unroll 1
        for (; i + U <= lane1; i += U) {
            double v[U];
#pragma unroll
            for (int j = 0; j < U; ++j) v[j] = add(i + j);
#pragma unroll
            for (int j = 0; j < U; j += 4) a += (v[j] + v[j + 1]) + (v[j + 2] + v[j + 3]);
        }
#pragma unroll 1
        for (; i < lane1; ++i) a += add(i);
        auto halves = [](double x, double y) { return make_uint4(__double2loint(x), __double2hiint(x), __double2loint(y), __double2hiint(y)); };
        if constexpr (KIND == kSumFirst) {
            // (the lanes' are put right when they are asked for)
            sh.lane_sum[warp][lane] = a;
            sh.lane_bend[warp][lane] = e;
            auto join = [&](const VerThree &v, bool is) {
                VerThree r;
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    const double x = ver_warp_sum(is ? __hiloint2double(v.v[j].y, v.v[j].x) : 0.0), y = ver_warp_sum(is ? __hiloint2double(v.v[j].w, v.v[j].z) : 0.0);
                    r.v[j] = halves(x, y);
                }
                return r;
            };
            const VerThree all = meet(join(VerThree{{halves(a, e), halves(b, d), halves(near, 0.0)}}, true), join);
#pragma unroll
            for (int j = 0; j < 3; ++j) found[2 * j] = __hiloint2double(all.v[j].y, all.v[j].x), found[2 * j + 1] = __hiloint2double(all.v[j].w, all.v[j].z);
        } else {
            sh.lane_sum[warp][lane] = a;
            auto join = [&](const VerOne &v, bool is) { return VerOne{{halves(ver_warp_sum(is ? __hiloint2double(v.v[0].y, v.v[0].x) : 0.0), 0.0)}}; };
            const uint4 all = meet(join(VerOne{{halves(a, 0.0)}}, true), join).v[0];
            found[0] = __hiloint2double(all.y, all.x);
        }
    };
    using First = std::integral_constant<int, kSumFirst>;
    using Left = std::integral_constant<int, kSumLeft>;
    using Target = std::integral_constant<int, kSumTarget>;

    int node = 0, level = 0, token = -1;
    bool mine_to_say = rank == 0;           // the CTA that knows the token behind
    // The row's children from row `from` on, one a lane, 32 at most (-1: none); from becomes where the next ones begin. Every warp looks by itself.
    auto children = [&](int &from) {
        if (!P.parents) {
            const int child = lane == 0 && from == node + 1 && from < n ? from : -1;
            from = n;
            return child;
        }
        int have = 0;
        __syncwarp();
        while (from < n && have < 32) {
            const unsigned kids = __ballot_sync(0xffffffffu, from + lane < n && sh.parents[from + lane] == node);
            const int at = have + __popc(kids & ((1u << lane) - 1u));
            const bool is = kids >> lane & 1u;
            if (is && at < 32) sh.kids[warp][at] = static_cast<int16_t>(from + lane);
            const unsigned late = __ballot_sync(0xffffffffu, is && at >= 32);
            have = min(32, have + __popc(kids));
            from += late ? __ffs(late) - 1 : 32;
        }
        from = min(from, n);
        __syncwarp();
        return lane < have ? static_cast<int>(sh.kids[warp][lane]) : -1;
    };
    for (;;) {
        if (tid == 0) sh.path[level] = static_cast<int16_t>(node);
        ++level;
        tp = target_row(node);
        int from = node + 1, child = children(from);
        dp = with_draft && __any_sync(0xffffffffu, child >= 0) ? draft_row(node) : nullptr;
        // the children's tokens and their logits are asked for beside the row
        int x = -1;
        float u = 0.0f, a = none, b = none;
        auto look_up = [&]() {
            x = child >= 0 ? P.tokens[f0 + child] : -1;
            u = child >= 0 ? P.uniforms[f0 + child] : 0.0f;
            const bool is = x >= 0 && x < vocab && !greedy;
            a = is ? static_cast<float>(tp[x]) : none;
            b = is && dp ? static_cast<float>(dp[x]) : none;
        };
        look_up();
        if constexpr (HELD) {
            int held = -1;
#pragma unroll
            for (int i = 0; i < kVerSlots; ++i)
                if (i < P.slots && slot_node[i] == node) held = i;
            if (held < 0) {                 // (none of those that were asked for: they are waited for, then their places are free)
                asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
                for (int i = 0; i < kVerSlots; ++i) slot_node[i] = -1;
                held = issued % P.slots;
                ask(node, dp != nullptr);
            }
            // those that may be next into the other places: of a chain the rows behind, of a tree the first child
            int newer = (issued - 1 - held) % P.slots;          // asked for behind this one
            const int kid = __shfl_sync(0xffffffffu, child, 0);
            while (newer < P.slots - 1) {
                const int next = P.parents ? (newer == 0 ? kid : -1) : node + 1 + newer < n ? node + 1 + newer : -1;
                if (next < 0) break;
                ask(next, with_draft && (P.parents || next + 1 < n));
                ++newer;
            }
            if (newer == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
            else if (newer == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else if (newer == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
            else asm volatile("cp.async.wait_group 3;" ::: "memory");
            __syncwarp();
            slot = held;
        }
        row_sums();
        if (gone || lost || !(sp.m < INFINITY)) break;
        if (greedy) {
            const int top = best;
            if (!(sp.s > none)) break;
            int to = -1;
            for (;;) {
                const unsigned hit = __ballot_sync(0xffffffffu, child >= 0 && x == top);
                if (hit) to = __shfl_sync(0xffffffffu, child, __ffs(hit) - 1);
                if (hit || from >= n) break;
                child = children(from);
                look_up();
            }
            if (to < 0) {
                token = top;
                break;
            }
            node = to;
            continue;
        }
        if (!(sp.s > 0.0f) || (dp && (!(sq.m < INFINITY) || !(sq.s > 0.0f)))) break;
        double left = 1.0, zp = 0.0, zq = 0.0, first_left = 0.0;          // S; the sums of the terms; S behind the first rejection
        bool exact = false;                 // the sums in 64 bits are known
        int to = -1;
        n_rejected = 0;
        c = bend = 0.0;
        for (;;) {
            // of each child: its probabilities, whether F32 can tell them, whether a brother in front has its token
            const bool is = x >= 0 && x < vocab;
            const float pa = (a - sp.m) * k, qb = (b - sq.m) * k;
            const float p = is && pa > -120.0f ? __fdividef(ver_ex2(pa), sp.s) : 0.0f, q = !dp ? 1.0f : is && qb > -120.0f ? __fdividef(ver_ex2(qb), sq.s) : 0.0f;
            const bool told = (pa > -120.0f || a == none) && (!dp || qb > -120.0f || b == none);
            unsigned todo = __ballot_sync(0xffffffffu, is);
            bool again = false;
            if (!dp && (todo & (todo - 1u))) again = (__match_any_sync(0xffffffffu, x) & ((1u << lane) - 1u)) != 0u;
            if (!dp && n_rejected > 0) again |= is_rejected(x);
            double exact_p = 0.0, exact_q = 1.0;
            auto make_exact = [&]() __attribute__((always_inline)) {
                if (!exact) {
                    double found[6];
                    if (dp) {
                        ratio = static_cast<double>(sp.s) / sq.s;
                        sums(First{}, found);
                        zp = found[2], zq = found[3];
                        bend = zp / zq - ratio;
                        over_zq = 1.0 / zq;
                        first_left = fmax(found[0] - bend * found[1], 0.0);
                        if (fabs(bend) * found[4] > 1e-13 * first_left || !(fabs(bend) <= 0x1p-19 * ratio)) {
                            ratio += bend;
                            bend = 0.0;
                            sums(Left{}, &first_left);
                        }
                        first_left /= zp;
                    } else {
                        const int held = n_rejected;
                        n_rejected = 0;     // (of all tokens)
                        sums(Target{}, found);
                        n_rejected = held;
                        zp = found[0];
                    }
                    over_zp = 1.0 / zp;
                    exact = true;
                }
                exact_p = is ? power(a, sp.m) * over_zp : 0.0;
                exact_q = dp ? (is ? power(b, sq.m) * over_zq : 0.0) : 1.0;
            };
            if (exact) make_exact();
            for (; todo; todo &= todo - 1u) {
                const int i = __ffs(todo) - 1;
                if (!dp && __shfl_sync(0xffffffffu, again, i)) continue;          // (nothing of it is left)
                // 1: taken, 2: F32 cannot tell
                const float l = u * static_cast<float>(left) * q;
                int verdict = exact || !told || !(fabsf(l - p) > P.unsure * (p + u * q)) ? 2 : l < p ? 1 : 0;
                verdict = __shfl_sync(0xffffffffu, verdict, i);
                if (verdict == 2) {
                    if (!exact) {
                        make_exact();
                        if (!dp) {          // (as the F32 tests took it, once more)
                            left = 1.0;
                            for (int j = 0; j < n_rejected; ++j) left -= power(static_cast<float>(tp[sh.rejected[j]]), sp.m) * over_zp;
                            left = fmax(left, 0.0);
                        }
                    }
                    verdict = __shfl_sync(0xffffffffu, static_cast<int>(u * left * exact_q < fmax(exact_p - c * exact_q, 0.0)), i);
                }
                if (verdict) {
                    to = __shfl_sync(0xffffffffu, child, i);
                    break;
                }
                if (dp) {
                    if (!exact) make_exact();
                    const bool second = c > 0.0;
                    c += left;
                    if (second) {
                        bend = 0.0;
                        ratio = c * zp * over_zq;
                        sums(Left{}, &left);
                        left *= over_zp;
                    } else {
                        left = first_left;
                    }
                } else {
                    left = fmax(left - (exact ? __shfl_sync(0xffffffffu, exact_p, i) : static_cast<double>(__shfl_sync(0xffffffffu, p, i))), 0.0);
                    const int out = __shfl_sync(0xffffffffu, x, i);
                    all_here();
                    if (tid == 0) sh.rejected[n_rejected] = out;
                    all_here();
                    if (lost) break;
                    ++n_rejected;
                }
            }
            if (to >= 0 || lost || from >= n) break;
            child = children(from);
            look_up();
        }
        if (to >= 0) {
            node = to;
            continue;
        }
        // ---- the token behind, from what is left
        double total = left * zp;
        const bool drawn_left = c > 0.0 && left > 0.0;
        if (!drawn_left) {                  // (nothing left: rounding; from p then)
            bend = 0.0;
            sums(Target{}, &total);
            if (!(total > 0.0)) {
                n_rejected = 0;
                sums(Target{}, &total);
            }
        }
        const double aim = static_cast<double>(P.uniforms[f0]) * total;
        double base = 0.0;
        // (behind the pass of the first rejection the sums of the terms that it left are beside)
        auto sum_in = [&](const uint4 &v, bool is) {
            const double sum = __hiloint2double(v.y, v.x);
            return !is ? 0.0 : bend != 0.0 ? fmax(sum - bend * __hiloint2double(v.w, v.z), 0.0) : sum;
        };
        if (ctas > 1) {
            const double v[1] = {sum_in(sh.slot[turn ^ 1][lane & (kVerCtas - 1)][0], lane < ctas)};
            const int owner = ver_pick(v, aim, base, lane);
            mine_to_say = max(owner, 0) == rank;
            if (gone || lost || !mine_to_say || owner < 0) break;
        }
        if (warp > 0) break;
        const double of_warp[1] = {sum_in(sh.warp_slot[turn ^ 1][lane & (kVerWarps - 1)][0], lane < kVerWarps)};
        const int w = max(ver_pick(of_warp, aim, base, lane), 0);
        const double of_lane[1] = {bend != 0.0 ? fmax(sh.lane_sum[w][lane] - bend * sh.lane_bend[w][lane], 0.0) : sh.lane_sum[w][lane]};
        const int l = max(ver_pick(of_lane, aim, base, lane), 0), begin = run_begin(rank * kVerWarps + w), last = min((l + 1) * piece, run_begin(rank * kVerWarps + w + 1) - begin);
        // that lane's piece, by a warp
        const T *px = run_of(0, w, begin), *qx = drawn_left ? run_of(1, w, begin) : nullptr;
#pragma unroll 1
        for (int i0 = l * piece; i0 < last; i0 += 32) {
            const int i = min(i0 + lane, last - 1);
            double v = drawn_left ? left_of(px, qx, i, ratio + bend) : power(static_cast<float>(px[i]), sp.m);
            if (i0 + lane >= last || (!drawn_left && n_rejected > 0 && is_rejected(begin + i))) v = 0.0;
            const double of_token[1] = {v}, in = ver_warp_sum(v);
            double at = base;
            const int found = ver_pick(of_token, aim, at, lane);
            if (found >= 0) token = begin + i0 + found;         // (what is found in front of the last ones stays where there is nothing behind it)
            if (base + in > aim) break;
            base += in;
        }
        break;
    }
    if constexpr (HELD) asm volatile("cp.async.wait_group 0;" ::: "memory");
    all_here();                             // (and the path is there)
    if (lost) {
        // None may leave while another one could send to it: those whose waits have run out meet here (of the others none sends any more: they have left), and wait once
        // more for what is on its way to them. Whatever the others said of the sequence before they left, it has no answer.
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
        ver_wait(&sh.full[turn ^ 1], (meetings - 1) >> 1 & 1);
        for (int i = tid; i < n; i += kVerThreads) P.path[f0 + i] = -1;
        if (tid == 0) P.count[seq] = P.next[seq] = -1;
        return;
    }
    if (mine_to_say && tid == 0) P.next[seq] = token;
    if (rank == 0) {
        if (tid == 0) P.count[seq] = level;
        for (int i = tid; i < n; i += kVerThreads) P.path[f0 + i] = i < level ? sh.path[i] : -1;
    }
}

// WD_VERIFY_STOP_AT=meeting[:CTA[:warp]] (tests): the wait of a sequence's CTAs for one another that runs out
struct VerStop {
    int at = -1, rank = -1, warp = -1;
    VerStop() {
        if (const char *v = std::getenv("WD_VERIFY_STOP_AT")) std::sscanf(v, "%d:%d:%d", &at, &rank, &warp);
    }
};

constexpr long long kVerHeld = 227 * 1024 - static_cast<long long>(sizeof(VerifyShared)) - 1024;         // bytes of rows that a CTA holds at most

template <class T, bool HELD, bool DRAFT>
int verify_launch(const VerifyParams &p, size_t smem, cudaStream_t s) {
    auto kernel = verify_kernel<T, HELD, DRAFT>;
    // (the attribute is the kernel's, for all threads: never what this call needs alone)
    if (HELD) WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kVerHeld)));
    if (p.ctas > 8) WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.n_seqs) * p.ctas);
    cfg.blockDim = dim3(kVerThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = p.ctas;
    a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    WD_TRY_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return WD_OK;
}
template <class T>
int verify_of(VerifyParams p, int n_sm, cudaStream_t s) {
    // A sequence's CTAs: enough that few sequences fill the SMs, none with less than four elements a thread.
    p.ctas = 1;
    while (p.ctas < kVerCtas && static_cast<long long>(p.n_seqs) * p.ctas * 2 <= 8 * n_sm && p.vocab >= p.ctas * 2 * kVerThreads * 4) p.ctas *= 2;
    p.piece = static_cast<int>((static_cast<long long>(p.vocab) + p.ctas * kVerThreads - 1) / (p.ctas * kVerThreads)) | 1;
    p.unsure = ver_unsure(p.piece);
    static const VerStop stop;
    p.stop_at = stop.at;
    p.stop_rank = stop.rank;
    p.stop_warp = stop.warp;
    // What shared memory holds of the rows: one row where there are more CTAs than SMs (up to 100 KB of it leave room for two of them an SM), up to four where there are fewer.
    const long long run_bytes = static_cast<long long>(p.piece) * 32 * sizeof(T) + 16, slot = run_bytes * kVerWarps * (p.draft ? 2 : 1);
    if (slot > kVerHeld) {
        p.slots = p.run_bytes = 0;
        return p.draft ? verify_launch<T, false, true>(p, 0, s) : verify_launch<T, false, false>(p, 0, s);
    }
    p.run_bytes = static_cast<int>(run_bytes);
    p.slots = static_cast<long long>(p.n_seqs) * p.ctas <= n_sm ? static_cast<int>(std::min<long long>(kVerSlots, kVerHeld / slot)) : 1;
    const size_t smem = static_cast<size_t>(slot) * p.slots;
    return p.draft ? verify_launch<T, true, true>(p, smem, s) : verify_launch<T, true, false>(p, smem, s);
}

}  // namespace
}  // namespace wd

extern "C" int wd_verify_drafts(const void *target_dev, const void *draft_dev, int type, int rows, int vocab, int64_t target_stride, int64_t draft_stride, int n_seqs,
                                const int *first_dev, const int *tokens_dev, const int *parents_dev, const float *uniforms_dev, const float *temperature_dev,
                                int *path_dev, int *count_dev, int *next_dev, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (type != WD_TYPE_F32 && type != WD_TYPE_F16 && type != WD_TYPE_BF16) return set_error(WD_E_INVALID, "verification: logits are F32, F16 or BF16");
        if (rows < 0 || vocab < 1 || n_seqs < 0 || rows > (1 << 30) || vocab > (1 << 30) || n_seqs > (1 << 24)) return set_error(WD_E_INVALID, "verification: rows, vocab and n_seqs");
        if (n_seqs == 0) return WD_OK;
        if (!first_dev && (rows % n_seqs || rows / n_seqs > wd::kVerRows)) return set_error(WD_E_INVALID, "verification: equal shares of at most 1024 rows");
        if (!count_dev || !next_dev || (rows > 0 && (!target_dev || !tokens_dev || !uniforms_dev || !path_dev))) return set_error(WD_E_INVALID, "null argument");
        const size_t size = type == WD_TYPE_F32 ? 4 : 2;
        if (reinterpret_cast<uintptr_t>(target_dev) % size || reinterpret_cast<uintptr_t>(draft_dev) % size) return set_error(WD_E_INVALID, "verification: logits are not aligned to their type");
        for (const void *p : {static_cast<const void *>(first_dev), static_cast<const void *>(tokens_dev), static_cast<const void *>(parents_dev), static_cast<const void *>(uniforms_dev),
                              static_cast<const void *>(temperature_dev), static_cast<const void *>(path_dev), static_cast<const void *>(count_dev), static_cast<const void *>(next_dev)})
            if (reinterpret_cast<uintptr_t>(p) % 4) return set_error(WD_E_INVALID, "verification: an argument is not aligned to its type");
        if (target_stride == 0) target_stride = vocab;
        if (draft_stride == 0) draft_stride = vocab;
        if (target_stride < vocab || (draft_dev && draft_stride < vocab)) return set_error(WD_E_INVALID, "verification: rows overlap");
        cudaPointerAttributes at{};
        const cudaError_t ce = cudaPointerGetAttributes(&at, rows > 0 ? target_dev : count_dev);
        if (ce != cudaSuccess || at.type == cudaMemoryTypeUnregistered || at.type == cudaMemoryTypeHost) {
            cudaGetLastError();
            return set_error(WD_E_INVALID, "verification: logits are not in device memory");
        }
        OnDevice on(at.device);
        if (!on.ok()) return set_error(WD_E_CUDA, "verification: the logits' device");
        int n_sm = 0;
        WD_TRY_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, at.device));
        wd::VerifyParams p{target_dev, draft_dev, target_stride, draft_stride, rows, vocab, n_seqs, 1, 0, 0, 1, first_dev, tokens_dev, parents_dev, uniforms_dev, temperature_dev,
                           path_dev, count_dev, next_dev};
        for (int i = 0; i < 32; ++i) p.power[i] = std::exp2(i / 32.0);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return type == WD_TYPE_F32 ? wd::verify_of<float>(p, n_sm, s) : type == WD_TYPE_F16 ? wd::verify_of<__half>(p, n_sm, s) : wd::verify_of<__nv_bfloat16>(p, n_sm, s);
    });
}
