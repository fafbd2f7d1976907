// Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits (wd_token_logprobs).
//
//   m = max x,  s = sum e^(x - m),  t = sum (x - m) e^(x - m):   log p = x - m - log s,   H = log s - t / s
//
// One pass over the logits, two CTAs an SM. A thread keeps its own m, s, t over rounds of 16 elements, which it copies into a ring of its own in shared
// memory, three rounds (F32; six of 16 bits) ahead and over the rows' ends too; it waits for no other thread between a row's first round and its end. A
// row is shared by the CTAs of a cluster where there are few rows (they meet in the first one's shared memory, so that no workspace is needed).
//
// The alternatives are collected beside: a key is (order of the value, lowest index first) in 64 bits, a candidate is what is not below the CTA's bar,
// and each warp has a list of candidates, which it cuts to its n_top best when it is full. The bar is the n_top-th of the maxima of groups of eight
// threads after the first round, and what one warp finds it to be after 2, 4, 8, ... rounds, so that few elements behind meet it, whatever their order; a
// warp that cuts its list raises it too.
//
// Bound: memory. 1,000 rows of 128,256 F32 with 20 alternatives: 114 us, 4.5 TB/s (a copy's rate: 80); what is missing goes to the candidates of a
// row's first rounds and to its end. Four rows of 151,936 with 5: 12 us of launch, the first bytes and the cluster's exchange.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "wd_device.cuh"
#include "wd_host.h"

namespace cg = cooperative_groups;
using wd_host::OnDevice;
using wd_host::set_error;

namespace wd {
namespace {

constexpr int kScoreThreads = 512, kScoreWarps = kScoreThreads / 32, kScoreTop = 32, kScoreOwn = 64, kScoreList = kScoreWarps * kScoreTop;
constexpr int kScoreRing = 12;              // 16 bytes of a thread's ring
typedef unsigned long long score_key;

struct ScoreParams {
    const void *logits;
    long long stride;
    int rows, vocab, n_top, ctas;
    const int *tokens;
    float *logprob, *entropy;
    int *top_ids;
    float *top_logprobs;
};

// larger values first, then lower indices; every key of a number is above 0
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);        // (-0 is 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ score_key key_of(float x, int i) { return static_cast<score_key>(order_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(i)); }

__device__ __forceinline__ float max_nan(float a, float b, float c) {        // a NaN stays one
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float ex2s(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int kN = 4;
    __device__ static void get(const uint4 &v, float *x) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
    __device__ static float one(const float *p) { return *p; }
};
template <>
struct Vec<__half> {
    static constexpr int kN = 8;
    __device__ static void get(const uint4 &v, float *x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    __device__ static float one(const __half *p) { return __half2float(*p); }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    __device__ static void get(const uint4 &v, float *x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    __device__ static float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
};

struct ScoreSums {
    float m, s, t, bad;         // s = sum 2^y, t = sum y 2^y, y = (x - m) log2 e; bad is not 0 for a row without a distribution
};
constexpr float kScoreLog2e = 1.44269504f, kScoreFloor = -3.402823466e38f;     // a maximum over nothing, and the lowest of a number
__device__ __forceinline__ ScoreSums both(const ScoreSums &a, const ScoreSums &b) {
    ScoreSums r;
    r.m = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - r.m) * kScoreLog2e, -200.0f), db = fmaxf((b.m - r.m) * kScoreLog2e, -200.0f), fa = ex2s(da), fb = ex2s(db);
    r.s = a.s * fa + b.s * fb;
    r.t = (a.t + da * a.s) * fa + (b.t + db * b.s) * fb;
    r.bad = a.bad + b.bad;
    return r;
}

struct ScoreShared {
    score_key own[kScoreWarps][kScoreOwn];          // the warps' candidates
    int own_count[kScoreWarps];
    score_key list[kScoreList], best[kScoreTop];    // the row's, at its end
    ScoreSums warp_sums[kScoreWarps], sums;
    __align__(16) uint32_t reached[kScoreThreads / 8];            // the groups' maxima, in order
    score_key others[8][kScoreTop];                 // of a cluster's first CTA: what the CTAs bring
    ScoreSums other_sums[8];
    int other_count[8];
    int count;
    score_key bar;
};

// The list is cut to its n best, in order. All threads; keys are distinct. A warp ranks a key: each lane compares it with some of the others.
__device__ __forceinline__ void score_cut(ScoreShared &sh, int n) {
    const int tid = threadIdx.x, lane = tid & 31, have = sh.count;
    for (int i = tid >> 5; i < have; i += kScoreWarps) {
        const score_key k = sh.list[i];
        int rank = 0;
        for (int j = 0; j < have; j += 32) rank += __popc(__ballot_sync(0xffffffffu, j + lane < have && sh.list[j + lane] > k));
        if (lane == 0 && rank < n) sh.best[rank] = k;
    }
    __syncthreads();
    const int left = min(have, n);
    if (tid < left) sh.list[tid] = sh.best[tid];
    if (tid == 0) sh.count = left;
    __syncthreads();
}
// A warp's candidates, `count` of them, are cut to their n best; where there are n the last of them is a bar for the row.
__device__ __forceinline__ int score_cut_own(score_key *own, int count, int n, score_key *bar, int lane) {
    __syncwarp();
    const score_key a = lane < count ? own[lane] : 0, b = lane + 32 < count ? own[lane + 32] : 0;
    int ra = 0, rb = 0;
    for (int j = 0; j < count; ++j) {
        const score_key k = own[j];
        ra += k > a;
        rb += k > b;
    }
    __syncwarp();
    if (a != 0 && ra < n) own[ra] = a;
    if (b != 0 && rb < n) own[rb] = b;
    __syncwarp();
    const int left = min(count, n);
    if (lane == 0 && left == n) atomicMax(bar, own[n - 1]);
    __syncwarp();
    return left;
}

template <class T>
__global__ void __launch_bounds__(kScoreThreads, 2) score_kernel(const __grid_constant__ ScoreParams P) {
    extern __shared__ __align__(128) uint8_t score_ring[];
    __shared__ ScoreShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = P.ctas, rank = ctas > 1 ? static_cast<int>(cluster.block_rank()) : 0, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_top = P.n_top;
    const int group = static_cast<int>(blockIdx.x) / ctas, groups = static_cast<int>(gridDim.x) / ctas;        // (blocks of a cluster follow one another)
    constexpr int VN = Vec<T>::kN, PER = 16 / VN, ROUND = kScoreThreads * PER, SLOTS = kScoreRing / PER;       // in 16 bytes: a thread, a round
    // Where a row's reads of 16 bytes are: from the first boundary on. What lies in front and behind are single elements of the first CTA's first round.
    struct Place {
        const T *x;
        int lead, n_vec, v0, v1;
    };
    auto place = [&](int row) {
        Place p;
        p.x = static_cast<const T *>(P.logits) + static_cast<size_t>(row) * P.stride;
        p.lead = min(static_cast<int>(((16u - static_cast<unsigned>(reinterpret_cast<uintptr_t>(p.x) & 15u)) & 15u) / sizeof(T)), P.vocab);
        p.n_vec = (P.vocab - p.lead) / VN;
        const int per_cta = (p.n_vec + ctas - 1) / ctas;
        p.v0 = min(rank * per_cta, p.n_vec);
        p.v1 = min(p.v0 + per_cta, p.n_vec);
        return p;
    };
    // the ring: rounds are asked for in the order in which they are read, one group of copies each (an empty one behind the last row)
    uint4 *ring = reinterpret_cast<uint4 *>(score_ring) + tid;
    int ask_row = group, ask_base = 0, ask_slot = 0;
    Place ask_at = place(group);
    ask_base = ask_at.v0;
    auto ask = [&]() {
        if (ask_row < P.rows) {
            const uint4 *xv = reinterpret_cast<const uint4 *>(ask_at.x + ask_at.lead) + ask_base + tid;
            const uint32_t to = smem_u32(ring + ask_slot * PER * kScoreThreads);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (ask_base + i * kScoreThreads + tid < ask_at.v1)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * kScoreThreads * 16), "l"(xv + i * kScoreThreads) : "memory");
            ask_base += ROUND;
            ask_slot = ask_slot + 1 == SLOTS ? 0 : ask_slot + 1;
            if (ask_base >= ask_at.v1 && (ask_row += groups) < P.rows) {
                ask_at = place(ask_row);
                ask_base = ask_at.v0;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < SLOTS; ++i) ask();
    int slot = 0;
#pragma unroll 1
    for (int row = group; row < P.rows; row += groups) {
        // Another CTA's shared memory is there from that CTA's start on: all of a cluster say here that they run, and wait for it in front of the exchange.
        if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
        const Place at = place(row);
        const T *x = at.x;
        const int lead = at.lead, tail0 = lead + at.n_vec * VN, loose = lead + P.vocab - tail0, v0 = at.v0, v1 = at.v1;
        ScoreSums mine = {kScoreFloor, 0.0f, 0.0f, 0.0f};
        if (tid == 0) {
            sh.count = 0;
            sh.bar = 1;
        }
        if (lane == 0) sh.own_count[warp] = 0;
        auto grow = [&](float top) {
            if (!(top < INFINITY)) mine.bad = 1.0f;
            if (top > mine.m) {
                const float d = fmaxf((mine.m - top) * kScoreLog2e, -200.0f), f = ex2s(d);
                mine.t = (mine.t + d * mine.s) * f;
                mine.s *= f;
                mine.m = top;
            }
        };
        auto add_clamped = [&](float x) {
            const float y = fmaxf((x - mine.m) * kScoreLog2e, -200.0f), e = ex2s(y);
            mine.s += e;
            mine.t = fmaf(e, y, mine.t);
        };
        // 16 elements. A logit of -inf, or one far under the maximum, makes 0 times -inf of a term; then the elements are added one by one.
        auto add = [&](const float *v, float top) {
            grow(top);
            float s = 0.0f, t = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = (v[i] - mine.m) * kScoreLog2e, e = ex2s(y);
                s += e;
                t = fmaf(e, y, t);
            }
            if (t == t) {
                mine.s += s;
                mine.t += t;
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) add_clamped(v[i]);
            }
        };
        // A lane's element joins its warp's candidates; false where they are full.
        auto join = [&](float v, int index) {
            const int at = atomicAdd(&sh.own_count[warp], 1);
            if (at < kScoreOwn) sh.own[warp][at] = key_of(v, index);
            return at < kScoreOwn;
        };
        // All lanes: the candidates are cut to their n best.
        auto make_room = [&]() {
            __syncwarp();
            const int left = score_cut_own(sh.own[warp], min(sh.own_count[warp], kScoreOwn), n_top, &sh.bar, lane);
            if (lane == 0) sh.own_count[warp] = left;
            __syncwarp();
        };
        auto bar_now = [&]() {          // (-inf is no candidate)
            const uint32_t least = static_cast<uint32_t>(*static_cast<volatile score_key *>(&sh.bar) >> 32);
            return least ? value_of(least) : -3.402823466e38f;
        };
        float given = NAN;          // the given token's logit
        if (rank == 0 && tid == 0 && P.logprob) {
            const int token = P.tokens[row];
            if (token >= 0 && token < P.vocab) given = Vec<T>::one(x + token);
        }
        float lone = -INFINITY;
        int lone_at = 0;
        const bool with_lone = rank == 0 && loose > 0;
        if (with_lone && tid < loose) {
            lone_at = tid < lead ? tid : tail0 + tid - lead;
            lone = Vec<T>::one(x + lone_at);
            grow(lone);
            add_clamped(lone);
        }
        __syncthreads();
        // The bar that the published maxima allow: the n_top-th of them. One warp, and the others may publish meanwhile: whatever it reads is an element
        // of its own for each group, and any n_top of those are reached by the least of them.
        auto raise = [&]() {
            const volatile uint32_t *o = sh.reached;
            const uint32_t a = o[lane], c = o[lane + 32];
            int ra = 0, rc = 0;
#pragma unroll 4
            for (int i = 0; i < 32; ++i) {
                const uint32_t x = __shfl_sync(0xffffffffu, a, i), y = __shfl_sync(0xffffffffu, c, i);
                ra += (x > a) + (y > a);
                rc += (x > c) + (y > c);
            }
            // those that fewer than n_top are above: the least of them
            const uint32_t least = __reduce_min_sync(0xffffffffu, min(ra < n_top ? a : 0xffffffffu, rc < n_top ? c : 0xffffffffu));
            if (lane == 0 && least != 0u) atomicMax(&sh.bar, static_cast<score_key>(least) << 32);
        };
#pragma unroll 1
        for (int base = v0, round = 1; base < v1 || round == 1; base += ROUND, ++round) {
            float v[16];
            asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
            const uint4 *from = ring + slot * PER * kScoreThreads;
            slot = slot + 1 == SLOTS ? 0 : slot + 1;
#pragma unroll
            for (int p = 0; p < PER; ++p) Vec<T>::get(from[p * kScoreThreads], v + p * VN);
            if (base + ROUND > v1) {        // the row's last round: what lies behind was not copied
#pragma unroll
                for (int p = 0; p < PER; ++p)
                    if (base + p * kScoreThreads + tid >= v1) {
#pragma unroll
                        for (int i = 0; i < VN; ++i) v[p * VN + i] = -INFINITY;
                    }
            }
            float top = v[0];
#pragma unroll
            for (int i = 1; i < 15; i += 2) top = max_nan(top, v[i], v[i + 1]);
            top = max_nan(top, v[15], v[15]);
            if (top > -INFINITY || top != top) add(v, top);
            if (n_top > 0) {
                unsigned late = 0;          // candidates that found no room
                if ((round & (round - 1)) == 0) {
                    uint32_t o = mine.s > 0.0f ? order_of(mine.m) : 0u;
                    o = max(o, __shfl_xor_sync(0xffffffffu, o, 1));
                    o = max(o, __shfl_xor_sync(0xffffffffu, o, 2));
                    o = max(o, __shfl_xor_sync(0xffffffffu, o, 4));
                    if ((lane & 7) == 0) sh.reached[tid >> 3] = o;
                    if (round == 1) {
                        __syncthreads();
                        if (warp == 0) raise();
                        __syncthreads();
                        if (lone >= bar_now()) join(lone, lone_at);          // (fewer than 32)
                    } else if (warp == (round >> 1) % kScoreWarps) {
                        raise();
                    }
                }
                const float bar_value = bar_now();
                if (top >= bar_value) {         // some lane now and then (a row with a NaN has no answer)
#pragma unroll
                    for (int i = 0; i < 16; ++i) late |= v[i] >= bar_value ? 1u << i : 0u;
#pragma unroll 1
                    while (late) {              // the values once more, from where they were copied to
                        const int i = __ffs(late) - 1;
                        const float y = Vec<T>::one(reinterpret_cast<const T *>(from + i / VN * kScoreThreads) + i % VN);
                        if (!join(y, lead + (base + i / VN * kScoreThreads + tid) * VN + i % VN)) break;
                        late &= late - 1;
                    }
                }
                while (__any_sync(0xffffffffu, late != 0u)) {
                    make_room();
                    const score_key bar = *static_cast<volatile score_key *>(&sh.bar);
                    while (late) {
                        const int i = __ffs(late) - 1, index = lead + (base + i / VN * kScoreThreads + tid) * VN + i % VN;
                        const float y = Vec<T>::one(reinterpret_cast<const T *>(from + i / VN * kScoreThreads) + i % VN);
                        if (key_of(y, index) >= bar && !join(y, index)) break;
                        late &= late - 1;
                    }
                }
            }
            ask();          // the slot has been read
        }
        // the CTA's sums and candidates
        auto over_lanes = [&](ScoreSums r) {
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const ScoreSums other = {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o), __shfl_xor_sync(0xffffffffu, r.t, o),
                                         __shfl_xor_sync(0xffffffffu, r.bad, o)};
                r = both(r, other);
            }
            return r;
        };
        mine = over_lanes(mine);
        if (lane == 0) sh.warp_sums[warp] = mine;
        __syncthreads();        // the bar is the row's last
        if (n_top > 0) {
            if (sh.own_count[warp] > kScoreTop) make_room();
            const score_key bar = sh.bar;
            for (int i = lane; i < min(sh.own_count[warp], kScoreOwn); i += 32) {
                const score_key k = sh.own[warp][i];
                if (k >= bar) sh.list[atomicAdd(&sh.count, 1)] = k;
            }
            __syncthreads();
            score_cut(sh, n_top);
        }
        const ScoreSums nothing = {kScoreFloor, 0.0f, 0.0f, 0.0f};
        if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (tid < 32) {
            const ScoreSums r = over_lanes(tid < kScoreWarps ? sh.warp_sums[tid] : nothing);
            if (tid == 0) {
                sh.sums = r;
                if (ctas > 1) {
                    ScoreShared *to = cluster.map_shared_rank(&sh, 0);
                    to->other_sums[rank] = r;
                    to->other_count[rank] = sh.count;
                }
            }
        }
        if (ctas > 1) {
            if (tid < sh.count) cluster.map_shared_rank(&sh, 0)->others[rank][tid] = sh.list[tid];
            cluster.sync();
        } else {
            __syncthreads();
        }
        if (rank == 0) {
            ScoreSums r = sh.sums;
            if (ctas > 1) {
                r = over_lanes(lane < ctas ? sh.other_sums[lane] : nothing);
                if (n_top > 0) {
                    if (tid >= n_top && tid < ctas * n_top && tid % n_top < sh.other_count[tid / n_top])        // (at most 8 x 32; the own ones are there)
                        sh.list[atomicAdd(&sh.count, 1)] = sh.others[tid / n_top][tid % n_top];
                    __syncthreads();
                    score_cut(sh, n_top);
                }
            }
            const bool none = r.bad != 0.0f || !(r.s > 0.0f);
            const float log_s = logf(r.s);
            if (tid == 0 && P.entropy) P.entropy[row] = none ? NAN : fmaxf(0.0f, log_s - 0.69314718f * (r.t / r.s));
            if (tid == 0 && P.logprob) P.logprob[row] = none ? NAN : (given - r.m) - log_s;
            if (tid < n_top) {
                const size_t to = static_cast<size_t>(row) * n_top + tid;
                const bool is = !none && tid < sh.count;
                const score_key k = is ? sh.list[tid] : 0;
                P.top_ids[to] = is ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)) : -1;
                P.top_logprobs[to] = none ? NAN : is ? (value_of(static_cast<uint32_t>(k >> 32)) - r.m) - log_s : -INFINITY;
            }
        }
        __syncthreads();        // what the next row begins with anew has been read (a cluster has no next row: its first CTA has one place for the others')
    }
}

template <class T>
int score_launch(ScoreParams p, int n_sm, cudaStream_t s) {
    // A row's CTAs: enough that few rows fill the SMs, none with less than a round.
    p.ctas = 1;
    while (p.ctas < 8 && static_cast<long long>(p.rows) * p.ctas * 2 <= 2 * n_sm && p.vocab >= p.ctas * 2 * kScoreThreads * 16) p.ctas *= 2;
    const int most = 2 * n_sm / p.ctas;         // groups of CTAs at once; a cluster has one row (p.rows * p.ctas <= 2 * n_sm)
    constexpr int smem = kScoreThreads * kScoreRing * 16;
    static_assert(2 * (smem + sizeof(ScoreShared) + 1024) <= 228 * 1024, "two CTAs an SM");
    WD_TRY_CUDA(cudaFuncSetAttribute(score_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows < most ? p.rows : most) * p.ctas);
    cfg.blockDim = dim3(kScoreThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = p.ctas;
    a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    WD_TRY_CUDA(cudaLaunchKernelEx(&cfg, score_kernel<T>, p));
    return WD_OK;
}

}  // namespace
}  // namespace wd

extern "C" int wd_token_logprobs(const void *logits_dev, int type, int rows, int vocab, int64_t stride, const int *tokens_dev, float *logprob_dev,
                                 float *entropy_dev, int n_top, int *top_ids_dev, float *top_logprobs_dev, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (type != WD_TYPE_F32 && type != WD_TYPE_F16 && type != WD_TYPE_BF16) return set_error(WD_E_INVALID, "token logprobs: logits are F32, F16 or BF16");
        if (rows < 0 || vocab < 1 || rows > (1 << 30) || vocab > (1 << 30)) return set_error(WD_E_INVALID, "token logprobs: rows and vocab");      // (sums of them stay in 32 bits)
        if (n_top < 0 || n_top > wd::kScoreTop) return set_error(WD_E_INVALID, "token logprobs: 0 to 32 alternatives");
        if (!logits_dev || (logprob_dev && !tokens_dev) || (n_top > 0 && (!top_ids_dev || !top_logprobs_dev)) || (!logprob_dev && !entropy_dev && n_top == 0))
            return set_error(WD_E_INVALID, "null argument");
        const size_t size = type == WD_TYPE_F32 ? 4 : 2;
        if (reinterpret_cast<uintptr_t>(logits_dev) % size) return set_error(WD_E_INVALID, "token logprobs: logits are not aligned to their type");
        if (stride == 0) stride = vocab;
        if (stride < vocab) return set_error(WD_E_INVALID, "token logprobs: rows overlap");
        if (rows == 0) return WD_OK;
        cudaPointerAttributes at{};
        const cudaError_t ce = cudaPointerGetAttributes(&at, logits_dev);
        if (ce != cudaSuccess || at.type == cudaMemoryTypeUnregistered || at.type == cudaMemoryTypeHost) {
            cudaGetLastError();
            return set_error(WD_E_INVALID, "token logprobs: logits are not in device memory");
        }
        OnDevice on(at.device);
        if (!on.ok()) return set_error(WD_E_CUDA, "token logprobs: the logits' device");
        int n_sm = 0;
        WD_TRY_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, at.device));
        wd::ScoreParams p{logits_dev, stride, rows, vocab, n_top, 1, tokens_dev, logprob_dev, entropy_dev, top_ids_dev, top_logprobs_dev};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return type == WD_TYPE_F32 ? wd::score_launch<float>(p, n_sm, s) : type == WD_TYPE_F16 ? wd::score_launch<__half>(p, n_sm, s) : wd::score_launch<__nv_bfloat16>(p, n_sm, s);
    });
}
