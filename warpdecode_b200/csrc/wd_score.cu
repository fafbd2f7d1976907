// Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits (wd_token_logprobs).
//
//   m = max x,  s = sum e^(x - m),  t = sum (x - m) e^(x - m):   log p = x - m - log s,   H = log s - t / s
//
// One pass over the logits. A CTA an SM walks over the rows, and a ring of bulk copies runs ahead of it, over the rows' ends too; a row is shared by
// the CTAs of a cluster where there are few rows (they meet in the first one's shared memory, so that no workspace is needed). A thread keeps its own
// m, s, t over rounds of 16 elements. The alternatives are collected beside: a key is (order of the value, lowest index first) in 64 bits, a candidate
// is what is not below the CTA's bar, and the bar comes from the first round (the n_top-th of the threads' maxima, to three bits behind the leading
// one) and rises when the list of candidates is cut to its n_top best. Behind the first rounds almost no element meets it.
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

constexpr int kScoreThreads = 1024, kScoreTop = 32, kScoreList = 1024, kScoreSlots = 6;
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

__device__ __forceinline__ float max_nan(float a, float b) {        // a NaN stays one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
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
    float m, s, t, bad;         // t in units of log 2: sum of y 2^y, y = (x - m) log2 e; bad is not 0 for a row without a distribution
};
constexpr float kScoreFloor = -3.0e38f;     // a maximum over nothing
__device__ __forceinline__ ScoreSums both(const ScoreSums &a, const ScoreSums &b) {
    ScoreSums r;
    r.m = fmaxf(a.m, b.m);
    const float da = (a.m - r.m) * 1.44269504f, db = (b.m - r.m) * 1.44269504f, fa = ex2s(fmaxf(da, -200.0f)), fb = ex2s(fmaxf(db, -200.0f));
    r.s = a.s * fa + b.s * fb;
    r.t = (fa > 0.0f ? (a.t + da * a.s) * fa : 0.0f) + (fb > 0.0f ? (b.t + db * b.s) * fb : 0.0f);
    r.bad = a.bad + b.bad;
    return r;
}

struct ScoreShared {
    score_key list[kScoreList], best[kScoreTop];
    ScoreSums warp_sums[kScoreThreads / 32], sums;
    float warp_max[kScoreThreads / 32];
    int count;
    score_key bar;
    uint64_t full[kScoreSlots];
};

// The list is cut to its n best, in order, and the bar set to the last of them where there are n. All threads; keys are distinct.
__device__ void score_cut(ScoreShared &sh, int n) {
    const int tid = threadIdx.x, have = min(sh.count, kScoreList);
    __syncthreads();
    for (int i = tid; i < have; i += kScoreThreads) {
        const score_key k = sh.list[i];
        int rank = 0;
        for (int j = 0; j < have; ++j) rank += sh.list[j] > k;
        if (rank < n) sh.best[rank] = k;
    }
    __syncthreads();
    const int left = min(have, n);
    if (tid < left) sh.list[tid] = sh.best[tid];
    if (tid == 0) {
        sh.count = left;
        if (left == n) sh.bar = max(sh.bar, sh.best[n - 1]);
    }
    __syncthreads();
}

template <class T>
constexpr int kSlotsOf = sizeof(T) == 4 ? 3 : kScoreSlots;        // 192 KB of a round's 16 elements a thread each

template <class T>
__global__ void __launch_bounds__(kScoreThreads, 1) score_kernel(const __grid_constant__ ScoreParams P) {
    extern __shared__ __align__(128) uint8_t score_ring[];
    __shared__ ScoreShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = P.ctas, rank = ctas > 1 ? static_cast<int>(cluster.block_rank()) : 0, tid = threadIdx.x, n_top = P.n_top;
    const int group = static_cast<int>(blockIdx.x) / ctas, groups = static_cast<int>(gridDim.x) / ctas;        // (blocks of a cluster follow one another)
    constexpr int VN = Vec<T>::kN, PER = 16 / VN, ROUND = kScoreThreads * PER, SLOTS = kSlotsOf<T>;      // elements of 16 bytes, 16 bytes of a thread and of a round
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
    // the ring: the first thread asks for rounds in the order in which they are read
    int ask_row = group, ask_base = -1, ask_slot = 0;
    auto ask = [&]() {
        while (ask_row < P.rows) {
            const Place p = place(ask_row);
            if (ask_base < 0) ask_base = p.v0;
            if (ask_base >= p.v1) {
                ask_row += groups;
                ask_base = -1;
                continue;
            }
            const uint32_t bytes = static_cast<uint32_t>(min(ROUND, p.v1 - ask_base)) * 16u;
            mbar_expect_tx(&sh.full[ask_slot], bytes);
            bulk_load(score_ring + static_cast<size_t>(ask_slot) * ROUND * 16, reinterpret_cast<const uint4 *>(p.x + p.lead) + ask_base, bytes, &sh.full[ask_slot]);
            ask_base += ROUND;
            ask_slot = ask_slot + 1 == SLOTS ? 0 : ask_slot + 1;
            return;
        }
    };
    if (tid == 0) {
        for (int i = 0; i < SLOTS; ++i) mbar_init(&sh.full[i], 1);
        mbar_fence_init();
        for (int i = 0; i < SLOTS; ++i) ask();
    }
    int slot = 0;
    uint32_t par = 0;
#pragma unroll 1
    for (int row = group; row < P.rows; row += groups) {
        const Place at_row = place(row);
        const T *x = at_row.x;
        const int lead = at_row.lead, tail0 = lead + at_row.n_vec * VN, loose = lead + P.vocab - tail0, v0 = at_row.v0, v1 = at_row.v1;
        if (tid == 0) {
            sh.count = 0;
            sh.bar = 1;
        }
        __syncthreads();
        ScoreSums mine = {kScoreFloor, 0.0f, 0.0f, 0.0f};
        auto add = [&](const float *v, int n, float top) {
            if (!(top < INFINITY)) mine.bad = 1.0f;
            if (top > mine.m) {
                const float d = (mine.m - top) * 1.44269504f, f = ex2s(fmaxf(d, -200.0f));
                mine.t = f > 0.0f ? (mine.t + d * mine.s) * f : 0.0f;
                mine.s *= f;
                mine.m = top;
            }
            float s = 0.0f, t = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n) {
                    const float y = fmaxf((v[i] - mine.m) * 1.44269504f, -200.0f), e = ex2s(y);
                    s += e;
                    t = fmaf(e, y, t);
                }
            mine.s += s;
            mine.t += t;
        };
        // candidates of a thread's elements; index(i) is the element's place in the row
        auto offer = [&](const float *v, int n, float top, auto index) {
            const score_key bar = sh.bar;
            if (order_of(top) < static_cast<uint32_t>(bar >> 32)) return;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n && v[i] > -INFINITY) {
                    const score_key k = key_of(v[i], index(i));
                    if (k >= bar) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < kScoreList) sh.list[at] = k;
                    }
                }
        };
        // after a round: a list that ran over is filled again above a higher bar, one that is half full is cut
        auto settle = [&](int before, auto again) {
            __syncthreads();
            int count = sh.count;
            __syncthreads();
            while (count > kScoreList) {
                // the n_top-th best of what found room is a bar that the round's and the older candidates can be held to
                const score_key keep = tid < before ? sh.list[tid] : 0;        // (before is at most kScoreList / 2, a thread for each)
                score_cut(sh, n_top);
                if (tid == 0) sh.count = 0;
                __syncthreads();
                if (keep != 0 && keep >= sh.bar) sh.list[atomicAdd(&sh.count, 1)] = keep;
                __syncthreads();
                before = sh.count;
                __syncthreads();
                again();
                __syncthreads();
                count = sh.count;
                __syncthreads();
            }
            if (count <= kScoreList / 2) return count;
            score_cut(sh, n_top);
            return min(count, n_top);
        };
        int before = 0;
        const int loose_n = rank == 0 ? loose : 0;
        float lone = -INFINITY;
        int lone_at = 0;
        if (tid < loose_n) {
            lone_at = tid < lead ? tid : tail0 + tid - lead;
            lone = Vec<T>::one(x + lone_at);
            add(&lone, 1, lone);
        }
        bool first = true;
#pragma unroll 1
        for (int base = v0; base < v1 || first; base += ROUND) {
            float v[16];
            if (base < v1) {
                // (a copy that never lands makes its row NaN)
                bool landed = false;
#pragma unroll 1
                for (unsigned i = 0; i < kSpinLimit && !landed; ++i) landed = mbar_try_wait(&sh.full[slot], par);
                if (!landed) mine.bad = 1.0f;
            }
            const uint4 *from = reinterpret_cast<const uint4 *>(score_ring + static_cast<size_t>(slot) * ROUND * 16) + tid;
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                if (base + p * kScoreThreads + tid < v1) {
                    Vec<T>::get(from[p * kScoreThreads], v + p * VN);
                } else {
#pragma unroll
                    for (int i = 0; i < VN; ++i) v[p * VN + i] = -INFINITY;
                }
            }
            const bool filled = base < v1;
            if (filled && ++slot == SLOTS) {
                slot = 0;
                par ^= 1;
            }
            float top = v[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = max_nan(top, v[i]);
            if (top > -INFINITY || top != top) add(v, 16, top);
            if (n_top > 0) {
                auto index = [&](int i) { return lead + (base + (i / VN) * kScoreThreads + tid) * VN + i % VN; };
                if (first) {
                    // the first bar: any value that at least n_top of the threads' maxima reach, as high as 12 halvings find
                    const float most = top == top ? fmaxf(top, lone) : lone;
                    const uint32_t o = most > -INFINITY ? order_of(most) : 0u;
                    uint32_t bar = 0;
                    for (int b = 31; b >= 20; --b) {
                        const uint32_t with = bar | 1u << b;
                        if (__syncthreads_count(o >= with) >= n_top) bar = with;
                    }
                    if (tid == 0) sh.bar = max(static_cast<score_key>(1), static_cast<score_key>(bar) << 32);
                    __syncthreads();
                }
                const bool with_lone = first && tid < loose_n;
                auto round = [&]() {
                    offer(v, 16, top, index);
                    if (with_lone) offer(&lone, 1, lone, [&](int) { return lone_at; });
                };
                round();
                before = settle(before, round);
            } else {
                __syncthreads();
            }
            if (tid == 0 && filled) ask();         // all threads have read the slot
            first = false;
        }
        // the CTA's sums
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const ScoreSums other = {__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.t, o),
                                     __shfl_xor_sync(0xffffffffu, mine.bad, o)};
            mine = both(mine, other);
        }
        if ((tid & 31) == 0) sh.warp_sums[tid >> 5] = mine;
        if (n_top > 0) score_cut(sh, n_top);
        __syncthreads();
        if (tid == 0) {
            ScoreSums r = sh.warp_sums[0];
            for (int w = 1; w < kScoreThreads / 32; ++w) r = both(r, sh.warp_sums[w]);
            sh.sums = r;
        }
        if (ctas > 1) cluster.sync();
        else __syncthreads();
        if (rank == 0) {
            ScoreSums r = sh.sums;
            for (int c = 1; c < ctas; ++c) r = both(r, *cluster.map_shared_rank(&sh.sums, c));
            if (n_top > 0 && ctas > 1) {
                // at most 16 x 32 candidates of the others go behind the own ones
                for (int i = tid; i < (ctas - 1) * n_top; i += kScoreThreads) {
                    ScoreShared *o = cluster.map_shared_rank(&sh, 1 + i / n_top);
                    if (i % n_top < o->count) sh.list[atomicAdd(&sh.count, 1)] = o->list[i % n_top];
                }
                __syncthreads();
                score_cut(sh, n_top);
            }
            const bool none = r.bad != 0.0f || !(r.s > 0.0f);
            const float log_s = logf(r.s);
            if (tid == 0 && P.entropy) P.entropy[row] = none ? NAN : fmaxf(0.0f, log_s - 0.69314718f * (r.t / r.s));
            if (tid == 0 && P.logprob) {
                const int token = P.tokens[row];
                P.logprob[row] = none || token < 0 || token >= P.vocab ? NAN : (Vec<T>::one(x + token) - r.m) - log_s;
            }
            if (tid < n_top) {
                const size_t to = static_cast<size_t>(row) * n_top + tid;
                const bool is = !none && tid < sh.count;
                const score_key k = is ? sh.list[tid] : 0;
                P.top_ids[to] = is ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)) : -1;
                P.top_logprobs[to] = none ? NAN : is ? (value_of(static_cast<uint32_t>(k >> 32)) - r.m) - log_s : -INFINITY;
            }
        }
        // the others' shared memory, and one's own, stay until they have been read
        if (ctas > 1) cluster.sync();
        else __syncthreads();
    }
}

template <class T>
int score_launch(ScoreParams p, int n_sm, cudaStream_t s) {
    // A row's CTAs: enough that few rows fill the SMs, none with less than a round.
    p.ctas = 1;
    while (p.ctas < 8 && static_cast<long long>(p.rows) * p.ctas * 2 <= n_sm && p.vocab >= p.ctas * 2 * kScoreThreads * 16) p.ctas *= 2;
    const int smem = kSlotsOf<T> * kScoreThreads * 16 * static_cast<int>(sizeof(T));
    WD_TRY_CUDA(cudaFuncSetAttribute(score_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows < n_sm / p.ctas ? p.rows : n_sm / p.ctas) * p.ctas);
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
        if (rows < 0 || vocab < 1) return set_error(WD_E_INVALID, "token logprobs: rows and vocab");
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
