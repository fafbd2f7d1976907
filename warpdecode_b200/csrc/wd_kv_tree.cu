// Attention over the 8-bit cache where the rows of each sequence are a tree of drafted tokens (wd_kv_attend_tree).
#include "wd_kv_launch.cuh"
#include "wd_kv_tree.cuh"

using namespace wd_kv;

namespace {

static_assert(wd::kTreeUnits * 128 <= 2 * wd::kAttMaxRows * wd::kAttWorkers * wd::kTreeUnits / 2, "the parts that a cache allocates");

// Which of the three kernels a step takes: the one that is expected to be through first, by what each was measured to take (us, d the head's size):
//   for few rows   11, and 1.2 (heads of 256 1.6) times what choose() counts
//   for trees      12 + d / 16 (F32 rows 3 more), and 0.85 + d^2 / 17,500 (F32 rows 1.3 times that) for 128 tokens by 128 rows and CTA; an item counts
//                  kTreeExtra tiles more, and the second kernel, which joins items that are cut, four
// (32 heads over 8 of 128, 16 sequences of 26 rows behind 300 to 6,000: 137 against 58 us; one of 13 rows behind 131: 12 against 16; 64 of 8 rows behind 90 to
// 3,000, of 64: 57 against 72.)
//   for prompts    11, and what choose() says, and a tenth of it all: it expands a tile of codes once for 256 rows of heads of up to 128 (64 rows behind 131,025, of 4 x 128: 184 us
//                  for 207 to 233), but gives sequences of other lengths no equal shares (16 sequences of 26 rows: 145 for 64)
enum TreeKernel { kFewRows, kTrees, kPairs };
struct TreeChoice {
    TreeKernel kernel;
    bool split;
};
TreeChoice choose_tree(const wd_kv_cache *c, bool f32, int window) {
    const int g = c->cfg.n_heads / c->cfg.n_kv_heads, d = c->cfg.head_dim, h = c->cfg.n_kv_heads, few_rows = d > 128 ? 8 : 16;
    double few = 0.0;
    long long items = 0, total = 0;
    int most = 0;
    for (int i = 0; i < c->book[0]; ++i) {
        const int *e = c->book.data() + wd::kKvHead + static_cast<size_t>(i) * wd::kKvStepWords;
        const long long rows = static_cast<long long>(e[2]) * g;
        if (rows == 0) continue;
        const int n = wd::tree_tiles(e[3], e[2], window, 128);
        const long long blocks = (rows + 127) / 128;
        few += static_cast<double>((rows + few_rows - 1) / few_rows) * h * 2 * n;
        items += blocks * h;
        total += blocks * h * (n + wd::kTreeExtra);
        most = std::max(most, n);
    }
    TreeChoice r;
    const long long chunk = wd::tree_chunk(total, c->n_sm, most, 128), whole = (items + c->n_sm - 1) / c->n_sm * (most + wd::kTreeExtra);
    r.split = whole > chunk + wd::kTreeExtra + 4;
    const double c_f = d / 36.0 * (f32 ? 1.2 : 1.0) * (d > 128 ? 0.4 : 1.2), c_t = (0.85 + d * d / 17500.0) * (f32 ? 1.3 : 1.0);
    const double of_few = 11.0 + c_f * few / (c->n_sm * (d > 128 ? 4.0 : 8.0)), of_tree = 12.0 + d / 16.0 + (f32 ? 3.0 : 0.0) + c_t * static_cast<double>(r.split ? chunk : whole);
    r.kernel = of_tree < of_few ? kTrees : kFewRows;
    if (d <= 128) {
        double of_pairs = 0.0;
        const bool split = choose(c, f32, window, true, &of_pairs).split;
        if (1.1 * (11.0 + of_pairs) < std::min(of_tree, of_few)) r = {kPairs, split};
    }
    return r;
}

template <int D, bool SPLIT>
int tree_launch(wd_kv_cache *c, const wd::KvTree &p, cudaStream_t s) {
    return by_codes(c, [&](auto e4m3) {
        using A = wd::TreePlan<D, SPLIT>;
        auto kernel = wd::kv_tree_kernel<D, SPLIT, decltype(e4m3)::value>;
        WD_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, A::kSmem));
        kernel<<<c->n_sm, wd::kPromptThreads, A::kSmem, s>>>(p);
        WD_TRY_CUDA(cudaGetLastError());
        if (!p.split) return WD_OK;
        cudaLaunchConfig_t cfg = {};            // (its blocks may take their places while the last CTAs of the first kernel work)
        cfg.gridDim = dim3(c->n_sm, 128 / wd::kTreeJoinRows<D>);
        cfg.blockDim = dim3(256);
        cfg.stream = s;
        cudaLaunchAttribute a[1];
        a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        a[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = a;
        cfg.numAttrs = 1;
        WD_TRY_CUDA(cudaLaunchKernelEx(&cfg, wd::kv_tree_join_kernel<D>, p));
        return WD_OK;
    });
}
template <int D>
int tree_of(wd_kv_cache *c, const wd::KvTree &p, bool pairs, cudaStream_t s) {
    if constexpr (D <= 128) {
        if (pairs) {
            wd::KvPromptTree r;
            static_cast<wd::KvPrompt &>(r) = p;
            r.parents = p.parents;
            return prompt_of<D>(c, r, s);
        }
    }
    return p.type == wd::kRowsF32 ? tree_launch<D, true>(c, p, s) : tree_launch<D, false>(c, p, s);
}

}  // namespace

extern "C" int wd_kv_attend_tree(wd_kv_cache *c, int layer, const void *q_dev, void *out_dev, const int *parents_dev, int type, float scale, int window, int64_t q_stride,
                                 int64_t out_stride, void *stream) {
    return wd_host::guarded([&]() -> int {
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        wd::KvAttendTree p;
        int rc = WD_OK;
        if (!attend_ready(c, layer, q_dev, out_dev, type, scale, window, q_stride, out_stride, s, p, rc)) return rc;
        if (!parents_dev || reinterpret_cast<uintptr_t>(parents_dev) % 4) return set_error(WD_E_INVALID, "key/value cache: parents are null, or not aligned to their type");
        if (c->max_rows > wd::kTreeRows) return set_error(WD_E_INVALID, "key/value cache: a tree has at most 128 rows");
        p.parents = parents_dev;
        OnDevice on(c->cfg.device);
        if (int r = note_capture(c, s)) return r;
        const TreeChoice by = choose_tree(c, p.type == wd::kRowsF32, p.window);
        if (by.kernel == kFewRows) return attend_few(c, p, s);
        const bool pairs = by.kernel == kPairs;
        c->last_kernel = pairs ? by.split ? "kv_prompt_kernel, kv_prompt_join_kernel" : "kv_prompt_kernel" : by.split ? "kv_tree_kernel, kv_tree_join_kernel" : "kv_tree_kernel";
        wd::KvTree r;
        fill_prompt(c, layer, p, by.split, &r);
        r.parents = parents_dev;
        r.cuts = reinterpret_cast<int4 *>(c->d_cta_part);
        switch (c->cfg.head_dim) {
            case 32: return tree_of<32>(c, r, pairs, s);
            case 64: return tree_of<64>(c, r, pairs, s);
            case 96: return tree_of<96>(c, r, pairs, s);
            case 128: return tree_of<128>(c, r, pairs, s);
            default: return tree_of<256>(c, r, pairs, s);
        }
    });
}
