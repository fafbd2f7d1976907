// Launches of attention over the 8-bit cache: which kernel a step takes, and its plan.
#pragma once

#include "wd_kv_attend.cuh"
#include "wd_kv_host.h"
#include "wd_kv_prompt.cuh"

namespace wd_kv {

// (P: wd::KvAttend, or wd::KvAttendTree)
template <int D, int N8, bool SPLIT, class P>
int attend_launch(wd_kv_cache *c, P &p, cudaStream_t s) {
    using A = wd::AttendPlan<D>;
    constexpr int kMost = 227 * 1024 - 8192 - (std::is_same_v<P, wd::KvAttendTree> ? 1024 : 0);      // what a block may have, less what the kernel declares itself
    static_assert(A::fixed_bytes(4, N8, SPLIT) + 4 * 2 * A::kSlot <= kMost, "four workers with two slots fit");
    // keys of one tile and values of the one before should be on their way while a worker computes
    for (p.workers = 8; p.workers > 4; p.workers /= 2)
        if ((kMost - A::fixed_bytes(p.workers, N8, SPLIT)) / (p.workers * A::kSlot) >= 3) break;
    p.slots = std::min(wd::kAttMaxSlots, (kMost - A::fixed_bytes(p.workers, N8, SPLIT)) / (p.workers * A::kSlot));
    const int smem = p.workers * p.slots * A::kSlot + A::fixed_bytes(p.workers, N8, SPLIT);
    return by_codes(c, [&](auto e4m3) {
        auto kernel = wd::kv_attend_kernel<D, N8, SPLIT, decltype(e4m3)::value, P>;
        WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<std::min(c->n_sm, wd::kAttMaxCtas), wd::kAttThreads, smem, s>>>(p);
        WD_TRY_CUDA(cudaGetLastError());
        return WD_OK;
    });
}
template <int D, class P>
int attend_of(wd_kv_cache *c, P &p, bool few, cudaStream_t s) {
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
// tree: of wd_kv_attend_tree, whose items see all of the step; us, where asked for: what the kernel for prompts is expected to take
inline Choice choose(const wd_kv_cache *c, bool f32, int window, bool tree = false, double *us = nullptr) {
    const int g = c->cfg.n_heads / c->cfg.n_kv_heads, d = c->cfg.head_dim, h = c->cfg.n_kv_heads;
    const int few_rows = d > 128 ? 8 : 16, item_rows = d > 128 ? 128 : 256;
    double few = 0.0, tiles = 0.0;
    long long items = 0;
    int most = 0;
    for (int i = 0; i < c->book[0]; ++i) {
        const int *e = c->book.data() + wd::kKvHead + static_cast<size_t>(i) * wd::kKvStepWords;
        const long long rows = static_cast<long long>(e[2]) * g;
        if (rows == 0) continue;
        const int seen = window ? std::min(e[3], window + (tree ? e[2] : item_rows / g)) : e[3], n = (seen + 127) / 128;
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
    if (us) *us = of_prompt;
    return r;
}

// (R: wd::KvPrompt, or wd::KvPromptTree)
template <int D, bool SPLIT, class R>
int prompt_launch(wd_kv_cache *c, const R &p, cudaStream_t s) {
    return by_codes(c, [&](auto e4m3) {
        auto kernel = wd::kv_prompt_kernel<D, SPLIT, decltype(e4m3)::value, R>;
        constexpr int smem = wd::PromptAttPlan<D, SPLIT>::kSmem;
        WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<c->n_sm, wd::kPromptThreads, smem, s>>>(p);
        if (p.split) wd::kv_prompt_join_kernel<D, R><<<2 * c->n_sm, 256, 0, s>>>(p);
        WD_TRY_CUDA(cudaGetLastError());
        return WD_OK;
    });
}
template <int D, class R>
int prompt_of(wd_kv_cache *c, const R &p, cudaStream_t s) {
    return p.type == wd::kRowsF32 ? prompt_launch<D, true>(c, p, s) : prompt_launch<D, false>(c, p, s);
}

// What attention calls check, and the launch of the kernel for few rows, p; rc is set where there is nothing more to do.
template <class P>
bool attend_ready(wd_kv_cache *c, int layer, const void *q_dev, void *out_dev, int type, float scale, int window, int64_t q_stride, int64_t out_stride, cudaStream_t s, P &p, int &rc) {
    auto check = [&]() -> int {
        if (int r = check_device(c)) return r;
        if (layer < 0 || layer >= c->cfg.n_layers) return set_error(WD_E_INVALID, "key/value cache: layer out of range");
        if (!(scale > 0.0f && scale * 1.4426950408889634 <= 3.4028234663852886e38)) return set_error(WD_E_INVALID, "key/value cache: the scale of the scores must be positive and finite");
        if (window < 0) return set_error(WD_E_INVALID, "key/value cache: a window is 0 (none) or at least 1");
        if (int r = rows_type(type, &p.type)) return r;
        if (c->book[0] == 0) return set_error(WD_E_STATE, "key/value cache: no step has begun");
        if (c->rows == 0) return check_not_captured(c, s);
        p.q_stride = q_stride;
        p.out_stride = out_stride;
        const long long width = static_cast<long long>(c->cfg.n_heads) * c->cfg.head_dim;
        if (int r = check_rows(q_dev, rows_size(p.type), &p.q_stride, width, "q")) return r;
        if (int r = check_rows(out_dev, rows_size(p.type), &p.out_stride, width, "out")) return r;
        if (q_dev == out_dev && p.q_stride != p.out_stride) return set_error(WD_E_INVALID, "key/value cache: out over q needs q's stride");
        return WD_OK;
    };
    rc = check();
    if (rc || c->rows == 0) return false;
    p.pool = c->d_pool + layer * c->pool_layer;
    p.scales = c->d_scales + layer * c->scales_layer;
    p.book = c->d_book;
    p.table = c->d_book + c->table_at;
    p.q = q_dev;
    p.out = out_dev;
    p.part = c->d_part;
    p.cta_part = c->d_cta_part;
    p.arrived = c->d_arrived;
    p.status = c->d_status;
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.window = window >= c->cfg.max_context ? 0 : window;
    p.max_seqs = c->cfg.max_seqs;
    p.vec = reinterpret_cast<uintptr_t>(q_dev) % 16 == 0 && p.q_stride * rows_size(p.type) % 16 == 0;
    p.s = c->shape;
    return true;
}
// the same for the kernels on tensor cores
inline void fill_prompt(const wd_kv_cache *c, int layer, const wd::KvAttend &p, bool split, wd::KvPrompt *r) {
    r->pool = p.pool, r->scales = p.scales, r->reach = c->d_reach + static_cast<size_t>(layer) * c->cfg.n_kv_heads, r->book = p.book, r->table = p.table, r->q = p.q, r->out = p.out;
    r->q_stride = p.q_stride, r->out_stride = p.out_stride, r->status = p.status, r->scale_log2 = p.scale_log2;
    r->type = p.type, r->window = p.window, r->s = p.s, r->part = c->d_part, r->ctas = c->n_sm;
    r->split = split;         // (the kernels count the items of the step that is current when they run)
    const size_t size = rows_size(p.type);
    r->vec = (reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out)) % 16 == 0 && p.q_stride * size % 16 == 0 && p.out_stride * size % 16 == 0;
}
template <class P>
int attend_few(wd_kv_cache *c, P &p, cudaStream_t s) {
    c->last_kernel = "kv_attend_kernel";
    const bool few = static_cast<long long>(c->max_rows) * (c->cfg.n_heads / c->cfg.n_kv_heads) <= 8;
    switch (c->cfg.head_dim) {
        case 32: return attend_of<32>(c, p, few, s);
        case 64: return attend_of<64>(c, p, few, s);
        case 96: return attend_of<96>(c, p, few, s);
        case 128: return attend_of<128>(c, p, few, s);
        default: return attend_of<256>(c, p, few, s);
    }
}

}  // namespace wd_kv
