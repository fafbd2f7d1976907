// Attention over the 8-bit cache where the rows of each sequence are a tree of drafted tokens (wd_kv_attend_tree): the kernels of wd_kv_attend, which look up a
// row's way to the root where a tile of tokens reaches into the step.
#include "wd_kv_launch.cuh"

using namespace wd_kv;

extern "C" int wd_kv_attend_tree(wd_kv_cache *c, int layer, const void *q_dev, void *out_dev, const int *parents_dev, int type, float scale, int window, int64_t q_stride,
                                 int64_t out_stride, void *stream) {
    return wd_host::guarded(
        [&]() -> int { return attend_call<wd::KvAttendTree, wd::KvPromptTree>(c, layer, q_dev, out_dev, parents_dev, type, scale, window, q_stride, out_stride, stream); });
}
