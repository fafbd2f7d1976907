// Launches of attention over the 8-bit cache: which kernel a step takes, and its plan.
#pragma once

#include "wd_kv_attend.cuh"
#include "wd_kv_host.h"
#include "wd_kv_prompt.cuh"

namespace wd_kv {

template <int D, int N8, bool SPLIT>
int attend_launch(wd_kv_cache *c, wd::KvAttend &p, cudaStream_t s) {
    using A = wd::AttendPlan<D>;
    constexpr int kMost = 227 * 1024 - 8192;        // what a block may have, less what the kernel declares itself
    static_assert(A::fixed_bytes(4, N8, SPLIT) + 4 * 2 * A::kSlot <= kMost, "four workers with two slots fit");
    // keys of one tile and values of the one before should be on their way while a worker computes
    for (p.workers = 8; p.workers > 4; p.workers /= 2)
        if ((kMost - A::fixed_bytes(p.workers, N8, SPLIT)) / (p.workers * A::kSlot) >= 3) break;
    p.slots = std::min(wd::kAttMaxSlots, (kMost - A::fixed_bytes(p.workers, N8, SPLIT)) / (p.workers * A::kSlot));
    const int smem = p.workers * p.slots * A::kSlot + A::fixed_bytes(p.workers, N8, SPLIT);
    return by_codes(c, [&](auto e4m3) {
        auto kernel = wd::kv_attend_kernel<D, N8, SPLIT, decltype(e4m3)::value>;
        WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<std::min(c->n_sm, wd::kAttMaxCtas), wd::kAttThreads, smem, s>>>(p);
        WD_TRY_CUDA(cudaGetLastError());
        return WD_OK;
    });
}
template <int D>
int attend_of(wd_kv_cache *c, wd::KvAttend &p, bool few, cudaStream_t s) {
    if constexpr (D > 128) few = true;       // (the sums of 16 rows of 256 do not fit a warp's registers)
    if (p.type == wd::kRowsF32) return few ? attend_launch<D, 1, true>(c, p, s) : attend_launch<D, (D > 128 ? 1 : 2), true>(c, p, s);
    return few ? attend_launch<D, 1, false>(c, p, s) : attend_launch<D, (D > 128 ? 1 : 2), false>(c, p, s);
}

// Which of the two attention kernels a step takes: the one that is expected to be through first, by what each was measured to take (us):
//   for few rows   c_f for 64 tokens of a head by 16 rows (8 of heads of 256) and worker: heads of 64 1.8, of 128 in F32 4.2, of 256 1.8
//   for prompts    3 more, and c_p for 128 tokens by 256 rows (128 of heads of 256) and CTA: heads of 64 1.8, of 128 in F32 3.4, of 256 4.2;
//                  8 more where items are cut into runs
// (64 rows a head of 64, 1,000 tokens: 15 against 23 us; 512 rows, 8,000 tokens: 63 against 39. Heads of 32 and 96 go by the lines through these points.)
struct Choice {
    bool prompt, split;
};
inline Choice choose(const wd_kv_cache *c, bool f32, int window) {
    const int g = c->cfg.n_heads / c->cfg.n_kv_heads, d = c->cfg.head_dim, h = c->cfg.n_kv_heads;
    const int few_rows = d > 128 ? 8 : 16, item_rows = d > 128 ? 128 : 256;
    double few = 0.0, tiles = 0.0;
    long long items = 0;
    int most = 0;
    for (int i = 0; i < c->book[0]; ++i) {
        const int *e = c->book.data() + wd::kKvHead + static_cast<size_t>(i) * wd::kKvStepWords;
        const long long rows = static_cast<long long>(e[2]) * g;
        if (rows == 0) continue;
        const int seen = window ? std::min(e[3], window + item_rows / g) : e[3], n = (seen + 127) / 128;
        const long long blocks = (rows + item_rows - 1) / item_rows;
        few += static_cast<double>((rows + few_rows - 1) / few_rows) * h * ((seen + 63) / 64);
        tiles += static_cast<double>(blocks) * h * n;
        items += blocks * h;
        most = std::max(most, n);
    }
    Choice r;
    const int runs = wd::prompt_runs(c->n_sm, items, most);
    r.split = runs > 1;
    const double c_f = d / 36.0 * (f32 ? 1.2 : 1.0) * (d > 128 ? 0.25 : 1.0), c_p = (1.0 + d / 80.0) * (f32 ? 1.3 : 1.0);
    const double of_few = c_f * few / (c->n_sm * (d > 128 ? 4.0 : 8.0));
    const double of_prompt = 3.0 + (r.split ? 8.0 + c_p * most / runs : c_p * std::max<double>(most, tiles / c->n_sm));
    r.prompt = of_prompt < of_few;
    return r;
}

template <int D, bool SPLIT>
int prompt_launch(wd_kv_cache *c, const wd::KvPrompt &p, cudaStream_t s) {
    return by_codes(c, [&](auto e4m3) {
        auto kernel = wd::kv_prompt_kernel<D, SPLIT, decltype(e4m3)::value>;
        constexpr int smem = wd::PromptAttPlan<D, SPLIT>::kSmem;
        WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<c->n_sm, wd::kPromptThreads, smem, s>>>(p);
        if (p.split) wd::kv_prompt_join_kernel<D><<<2 * c->n_sm, 256, 0, s>>>(p);
        WD_TRY_CUDA(cudaGetLastError());
        return WD_OK;
    });
}
template <int D>
int prompt_of(wd_kv_cache *c, const wd::KvPrompt &p, cudaStream_t s) {
    return p.type == wd::kRowsF32 ? prompt_launch<D, true>(c, p, s) : prompt_launch<D, false>(c, p, s);
}

}  // namespace wd_kv
