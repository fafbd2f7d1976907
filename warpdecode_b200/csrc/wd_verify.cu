// Verification of drafted tokens against the target's probabilities, from given random numbers (wd_verify_drafts).
//
// p = softmax(x / T), q the draft's. At a row whose children were drawn from q, what is left of p after j rejections is proportional to max(p - c_j q, 0):
//   c_0 = 0,  S(c) = sum max(p - c q, 0),  c_(j + 1) = c_j + S(c_j)
// (one rejection makes max(r - q, 0) / Z of r = max(p - c q, 0) / S, and max(max(p - c q, 0) / S - q, 0) S = max(p - (c + S) q, 0)), so that nothing of the
// vocabulary's size is kept from one child to the next, and a number each decides: u S q(x) < max(p(x) - c q(x), 0).
//
// A cluster of CTAs goes down a sequence's tree and reads the rows on its way alone, not those of all drafts. A row's maximum and sum are F32 and decide
// for a child that is not within 1e-4 of its border. What is nearer, and every draw, is made of sums in 64 bits: the running sums of 150,000 tokens lie 1e-7
// apart where the unlikely ones are, and the heavy ones' F32 errors (3e-8) would choose among them. The CTAs meet in their shared memories: each brings its
// sums to all, and all come to the same decision by the same arithmetic, so that nothing is sent back.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "wd_device.cuh"
#include "wd_host.h"

namespace cg = cooperative_groups;
using wd_host::OnDevice;
using wd_host::set_error;

namespace wd {
namespace {

constexpr int kVerThreads = 512, kVerWarps = kVerThreads / 32, kVerCtas = 16, kVerRows = 1024;
constexpr float kVerGreedy = 1e-6f, kVerFloor = -3.402823466e38f;
constexpr double kVerUnsure = 1e-4;        // F32 sums and exponentials are off by less than half of it

struct VerifyParams {
    const void *target, *draft;
    long long target_stride, draft_stride;
    int rows, vocab, n_seqs, ctas;
    const int *first, *tokens, *parents;
    const float *uniforms, *temperature;
    int *path, *count, *next;
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

template <class T>
struct Elements {
    static constexpr int kN = 16 / sizeof(T);
    __device__ static void get(const uint4 &v, float *x) {
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int i = 0; i < kN; ++i) x[i] = static_cast<float>(e[i]);
    }
};

struct RowSum {             // s = sum 2^(k (x - m)); m is a NaN or +inf where the row has no distribution
    float m, s;
};
__device__ __forceinline__ RowSum joined(RowSum a, RowSum b, float k) {
    RowSum r;
    r.m = ver_max(a.m, b.m);
    r.s = a.s * ver_ex2(fmaxf((a.m - r.m) * k, -200.0f)) + b.s * ver_ex2(fmaxf((b.m - r.m) * k, -200.0f));
    return r;
}
// larger values first, then lower indices
__device__ __forceinline__ unsigned long long ver_key(float x, int i) {
    const uint32_t b = __float_as_uint(x + 0.0f), o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return static_cast<unsigned long long>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}

struct VerifyShared {
    double slot[2][kVerCtas][2];            // what the CTAs of a cluster bring, in turn
    RowSum row_slot[2][kVerCtas][2];
    unsigned long long key_slot[2][kVerCtas];
    RowSum warp_row[2][kVerWarps];
    unsigned long long warp_key[kVerWarps];
    double warp_sum[2][kVerWarps];
    int rejected[kVerRows];                 // tokens
    int last;
};

enum { kSumBoth, kSumLeft, kSumTarget };    // of p and of q; of max(p - c q, 0); of p without the rejected tokens

template <class T>
__global__ void __launch_bounds__(kVerThreads) verify_kernel(const __grid_constant__ VerifyParams P) {
    __shared__ VerifyShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = P.ctas, rank = ctas > 1 ? static_cast<int>(cluster.block_rank()) : 0, seq = static_cast<int>(blockIdx.x) / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = P.vocab;
    const int share = P.rows / P.n_seqs;
    const int f0 = P.first ? min(max(P.first[seq], 0), P.rows) : seq * share, f1 = P.first ? min(max(P.first[seq + 1], f0), P.rows) : f0 + share, n = f1 - f0;
    if (n == 0 || n > kVerRows) {
        if (rank == 0) {
            for (int i = tid; i < n; i += kVerThreads) P.path[f0 + i] = -1;
            if (tid == 0) P.count[seq] = 0, P.next[seq] = -1;
        }
        return;
    }
    if (ctas > 1) cluster.sync();           // another CTA's shared memory is there from its start on
    const float heat = P.temperature ? P.temperature[seq] : 1.0f;
    const bool greedy = !(heat >= kVerGreedy);
    const float k = greedy ? 1.44269504f : static_cast<float>(1.4426950408889634 / heat);
    const double inv_heat = greedy ? 1.0 : 1.0 / heat;
    int turn = 0;                           // of the slots

    const T *tp = nullptr, *dp = nullptr;   // the row's logits; of the draft: null where it is not asked
    RowSum sp{}, sq{};
    unsigned long long best = 0;
    // maxima and sums of the row, or its largest logit
    auto row_sums = [&]() {
        constexpr int VN = Elements<T>::kN, U = 4;
        RowSum mine[2] = {{kVerFloor, 0.0f}, {kVerFloor, 0.0f}};
        unsigned long long key = 0;
        int lead[2], n_vec[2], v0[2], v1[2];
        const T *x[2] = {tp, dp};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            lead[w] = min(static_cast<int>(((16u - static_cast<unsigned>(reinterpret_cast<uintptr_t>(x[w]) & 15u)) & 15u) / sizeof(T)), vocab);
            n_vec[w] = x[w] ? (vocab - lead[w]) / VN : 0;
            const int per = (n_vec[w] + ctas - 1) / ctas;
            v0[w] = min(rank * per, n_vec[w]);
            v1[w] = min(v0[w] + per, n_vec[w]);
        }
        auto add = [&](int w, const float *v, int count, int at) {
            float top = v[0];
            for (int i = 1; i < count; ++i) top = ver_max(top, v[i]);
            if (greedy) {
                mine[w].m = ver_max(mine[w].m, top);
                const uint32_t seen = static_cast<uint32_t>(key >> 32);
                if (static_cast<uint32_t>(ver_key(top, 0) >> 32) > seen) {          // (of equals the one met first has the lowest index)
                    for (int i = 0; i < count; ++i) key = max(key, ver_key(v[i], at + i));
                }
                return;
            }
            RowSum &r = mine[w];
            const float now = ver_max(r.m, top);
            float s = r.s * ver_ex2(fmaxf((r.m - now) * k, -200.0f));
            for (int i = 0; i < count; ++i) s += ver_ex2(fmaxf((v[i] - now) * k, -200.0f));
            r.m = now, r.s = s;
        };
        for (int base = tid; base < max(v1[0] - v0[0], v1[1] - v0[1]); base += U * kVerThreads) {
            uint4 u[2][U];
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (v0[w] + base + i * kVerThreads < v1[w]) u[w][i] = __ldg(reinterpret_cast<const uint4 *>(x[w] + lead[w]) + v0[w] + base + i * kVerThreads);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (v0[w] + base + i * kVerThreads < v1[w]) {
                        float v[VN];
                        Elements<T>::get(u[w][i], v);
                        add(w, v, VN, lead[w] + (v0[w] + base + i * kVerThreads) * VN);
                    }
        }
        if (rank == 0) {                    // what lies in front of the first boundary of 16 bytes, and behind the last
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int tail = lead[w] + n_vec[w] * VN, loose = x[w] ? lead[w] + vocab - tail : 0;
                if (tid < loose) {
                    const int i = tid < lead[w] ? tid : tail + tid - lead[w];
                    const float v = static_cast<float>(x[w][i]);
                    add(w, &v, 1, i);
                    if (greedy && w == 0) key = max(key, ver_key(v, i));
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
#pragma unroll
            for (int w = 0; w < 2; ++w) mine[w] = joined(mine[w], RowSum{__shfl_xor_sync(0xffffffffu, mine[w].m, o), __shfl_xor_sync(0xffffffffu, mine[w].s, o)}, k);
            key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        }
        if (lane == 0) sh.warp_row[0][warp] = mine[0], sh.warp_row[1][warp] = mine[1], sh.warp_key[warp] = key;
        __syncthreads();
        if (warp == 0) {
            mine[0] = mine[1] = RowSum{kVerFloor, 0.0f};
            key = 0;
            if (lane < kVerWarps) mine[0] = sh.warp_row[0][lane], mine[1] = sh.warp_row[1][lane], key = sh.warp_key[lane];
#pragma unroll
            for (int o = 16; o; o >>= 1) {
#pragma unroll
                for (int w = 0; w < 2; ++w) mine[w] = joined(mine[w], RowSum{__shfl_xor_sync(0xffffffffu, mine[w].m, o), __shfl_xor_sync(0xffffffffu, mine[w].s, o)}, k);
                key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
            }
            if (lane < ctas) {
                VerifyShared *to = ctas > 1 ? cluster.map_shared_rank(&sh, lane) : &sh;
                to->row_slot[turn][rank][0] = mine[0];
                to->row_slot[turn][rank][1] = mine[1];
                to->key_slot[turn][rank] = key;
            }
        }
        if (ctas > 1) cluster.sync();
        else __syncthreads();
        sp = sq = RowSum{kVerFloor, 0.0f};
        best = 0;
        for (int r = 0; r < ctas; ++r) {
            sp = joined(sp, sh.row_slot[turn][r][0], k);
            sq = joined(sq, sh.row_slot[turn][r][1], k);
            best = max(best, sh.key_slot[turn][r]);
        }
        turn ^= 1;
    };

    // ---- in 64 bits: a warp has an even run of the vocabulary, the warps of a CTA and the CTAs one behind the other
    const int run = ((vocab + ctas * kVerWarps - 1) / (ctas * kVerWarps) + 31) / 32 * 32;
    const long long run0 = static_cast<long long>(rank * kVerWarps + warp) * run;
    double zp = 0.0, zq = 0.0, c = 0.0;
    int n_rejected = 0, kind = kSumBoth;
    auto power = [&](const T *x, float m, long long i) {
        const float v = static_cast<float>(x[i]);
        return v == -INFINITY ? 0.0 : exp((static_cast<double>(v) - static_cast<double>(m)) * inv_heat);
    };
    // what token i adds to a sum
    auto weight = [&](long long i, double &second) {
        double w = power(tp, sp.m, i);
        if (kind == kSumTarget) {
            for (int j = 0; j < n_rejected; ++j)
                if (sh.rejected[j] == i) w = 0.0;
        } else if (kind == kSumLeft) {
            w = fmax(w / zp - c * (power(dp, sq.m, i) / zq), 0.0);
        } else if (dp) {
            second += power(dp, sq.m, i);
        }
        return w;
    };
    int sums_turn = 0;
    auto sums = [&](int which, double &first, double &second) {
        kind = which;
        double a = 0.0, b = 0.0;
        const long long end = min(run0 + run, static_cast<long long>(vocab));
#pragma unroll 4
        for (long long i = run0 + lane; i < end; i += 32) a += weight(i, b);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        __syncthreads();                    // (what an earlier turn left has been read)
        if (lane == 0) sh.warp_sum[0][warp] = a, sh.warp_sum[1][warp] = b;
        __syncthreads();
        if (warp == 0 && lane < ctas) {
            a = b = 0.0;
            for (int w = 0; w < kVerWarps; ++w) a += sh.warp_sum[0][w], b += sh.warp_sum[1][w];
            VerifyShared *to = ctas > 1 ? cluster.map_shared_rank(&sh, lane) : &sh;
            to->slot[turn][rank][0] = a;
            to->slot[turn][rank][1] = b;
        }
        if (ctas > 1) cluster.sync();
        else __syncthreads();
        first = second = 0.0;
        for (int r = 0; r < ctas; ++r) first += sh.slot[turn][r][0], second += sh.slot[turn][r][1];
        sums_turn = turn;
        turn ^= 1;
    };

    int node = 0, level = 0, token = -1;
    bool mine_to_say = rank == 0;           // the CTA that knows the token behind
    for (;;) {
        const int row = f0 + node;
        if (rank == 0 && tid == 0) P.path[f0 + level] = node;
        ++level;
        // the row's next child behind `after`; every warp looks by itself
        auto child_behind = [&](int after) {
            if (!P.parents) return after == node && node + 1 < n ? node + 1 : n;
            for (int i = after + 1; i < n; i += 32) {
                const unsigned there = __ballot_sync(0xffffffffu, i + lane < n && P.parents[f0 + i + lane] == node);
                if (there) return i + __ffs(there) - 1;
            }
            return n;
        };
        int child = child_behind(node);
        tp = static_cast<const T *>(P.target) + static_cast<size_t>(row) * P.target_stride;
        dp = P.draft && !greedy && child < n ? static_cast<const T *>(P.draft) + static_cast<size_t>(row) * P.draft_stride : nullptr;
        row_sums();
        if (!(sp.m < INFINITY) || (greedy ? !(sp.m > -INFINITY) || best <= ver_key(-INFINITY, 0) : !(sp.s > 0.0f)) || (dp && (!(sq.m < INFINITY) || !(sq.s > 0.0f)))) break;
        int to = -1;
        if (greedy) {
            const int top = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
            for (; child < n; child = child_behind(child))
                if (P.tokens[f0 + child] == top) {
                    to = child;
                    break;
                }
            if (to < 0) {
                token = top;
                break;
            }
            node = to;
            continue;
        }
        double left = 1.0;                  // S
        bool exact = false;                 // the sums in 64 bits are known
        n_rejected = 0;
        c = 0.0;
        auto make_exact = [&]() {
            if (!exact) sums(kSumBoth, zp, zq);
            exact = true;
        };
        for (; child < n; child = child_behind(child)) {
            const int x = P.tokens[f0 + child];
            if (x < 0 || x >= vocab) continue;
            const double u = P.uniforms[f0 + child];
            bool again = false;
            for (int j = 0; j < n_rejected; ++j) again |= sh.rejected[j] == x;
            bool taken = false, sure = false;
            if (!exact) {
                const float a = static_cast<float>(tp[x]), b = dp ? static_cast<float>(dp[x]) : 0.0f;
                const float pa = (a - sp.m) * k, qb = dp ? (b - sq.m) * k : 0.0f;
                const double p = pa > -120.0f ? static_cast<double>(ver_ex2(pa)) / sp.s : 0.0, q = dp ? (qb > -120.0f ? static_cast<double>(ver_ex2(qb)) / sq.s : 0.0) : 1.0;
                const double l = u * left * q;
                sure = (pa > -120.0f || a == -INFINITY) && (qb > -120.0f || b == -INFINITY) && fabs(l - p) > kVerUnsure * (p + u * q);
                taken = l < p;
                if (!dp && !taken && sure && !again) left = fmax(left - p, 0.0);
            }
            if (!sure) {
                make_exact();
                const double p = power(tp, sp.m, x) / zp, q = dp ? power(dp, sq.m, x) / zq : 1.0;
                if (!dp) {
                    left = 1.0;
                    for (int j = 0; j < n_rejected; ++j) left -= power(tp, sp.m, sh.rejected[j]) / zp;
                    left = fmax(left, 0.0);
                }
                taken = u * left * q < fmax(p - c * q, 0.0);
            }
            if (!dp) taken = taken && !again;
            if (taken) {
                to = child;
                break;
            }
            if (dp) {
                make_exact();
                c += left;
                double none;
                sums(kSumLeft, left, none);
            } else if (!again) {
                __syncthreads();
                if (tid == 0) sh.rejected[n_rejected] = x;
                __syncthreads();
                ++n_rejected;
            }
        }
        if (to >= 0) {
            node = to;
            continue;
        }
        // ---- the token behind, from what is left
        double total = left, none;
        if (c == 0.0 || !(left > 0.0)) {    // (nothing left: rounding; from p then)
            sums(kSumTarget, total, none);
            if (!(total > 0.0)) {
                n_rejected = 0;
                sums(kSumTarget, total, none);
            }
        }
        const double aim = static_cast<double>(P.uniforms[f0]) * total;
        // the first of `count` sums whose running sum is above the aim, or the last one that is not 0; `base`: of those in front of it
        auto first_above = [&](auto sum, int count, double &base) {
            int last = 0;
            double at = base, last_base = base;
            for (int i = 0; i < count; ++i) {
                const double s = sum(i);
                if (s > 0.0) {
                    last = i, last_base = at;
                    if (at + s > aim) break;
                }
                at += s;
            }
            base = last_base;
            return last;
        };
        double base = 0.0;
        const int owner = first_above([&](int r) { return sh.slot[sums_turn][r][0]; }, ctas, base);
        mine_to_say = owner == rank;
        if (!mine_to_say) break;
        const int w0 = first_above([&](int w) { return sh.warp_sum[0][w]; }, kVerWarps, base);
        const long long start = static_cast<long long>(rank * kVerWarps + w0) * run, end = min(start + run, static_cast<long long>(vocab));
        // that warp's run, by all of the CTA's: 32 tokens a warp at a time
        if (tid == 0) sh.last = -1;
        token = -1;
        for (long long i0 = start; i0 < end && token < 0; i0 += kVerThreads) {
            const long long i = i0 + tid;
            double unused = 0.0;
            const double w = i < end ? weight(i, unused) : 0.0;
            double upto = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            __syncthreads();
            if (lane == 31) sh.warp_sum[1][warp] = upto;
            if (w > 0.0) atomicMax(&sh.last, static_cast<int>(i));
            __syncthreads();
            double at = base;
            for (int v = 0; v < warp; ++v) at += sh.warp_sum[1][v];
            const unsigned above = __ballot_sync(0xffffffffu, w > 0.0 && at + upto > aim);
            __syncthreads();
            if (lane == 0) sh.warp_key[warp] = above ? static_cast<unsigned long long>(i0 + warp * 32 + __ffs(above) - 1) : ~0ull;
            __syncthreads();
            for (int v = 0; v < kVerWarps && token < 0; ++v)
                if (sh.warp_key[v] != ~0ull) token = static_cast<int>(sh.warp_key[v]);
            for (int v = 0; v < kVerWarps; ++v) base += sh.warp_sum[1][v];
        }
        if (token < 0) token = sh.last;
        break;
    }
    if (mine_to_say && tid == 0) P.next[seq] = token;
    if (rank == 0) {
        if (tid == 0) P.count[seq] = level;
        for (int i = level + tid; i < n; i += kVerThreads) P.path[f0 + i] = -1;
    }
}

template <class T>
int verify_launch(VerifyParams p, int n_sm, cudaStream_t s) {
    // A sequence's CTAs: enough that few sequences fill the SMs, none with less than two elements a thread.
    p.ctas = 1;
    while (p.ctas < kVerCtas && static_cast<long long>(p.n_seqs) * p.ctas * 2 <= 4 * n_sm && p.vocab >= p.ctas * 2 * kVerThreads * 2) p.ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.n_seqs) * p.ctas);
    cfg.blockDim = dim3(kVerThreads);
    cfg.stream = s;
    cudaLaunchAttribute a[1];
    a[0].id = cudaLaunchAttributeClusterDimension;
    a[0].val.clusterDim.x = p.ctas;
    a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
    cfg.attrs = a;
    cfg.numAttrs = 1;
    if (p.ctas > 8) WD_TRY_CUDA(cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    WD_TRY_CUDA(cudaLaunchKernelEx(&cfg, verify_kernel<T>, p));
    return WD_OK;
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
        wd::VerifyParams p{target_dev, draft_dev, target_stride, draft_stride, rows, vocab, n_seqs, 1, first_dev, tokens_dev, parents_dev, uniforms_dev, temperature_dev,
                           path_dev, count_dev, next_dev};
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return type == WD_TYPE_F32 ? wd::verify_launch<float>(p, n_sm, s) : type == WD_TYPE_F16 ? wd::verify_launch<__half>(p, n_sm, s) : wd::verify_launch<__nv_bfloat16>(p, n_sm, s);
    });
}
