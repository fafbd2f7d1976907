// Host side of the 8-bit key/value cache (wd_kv_*): which sequence holds which pages, the step, and the launches.
#include <algorithm>
#include <cmath>
#include <climits>
#include <memory>
#include <type_traits>
#include <cstring>
#include <unordered_map>
#include <vector>

#include "wd_host.h"
#include "wd_kv_attend.cuh"
#include "wd_kv_kernels.cuh"
#include "wd_kv_prompt.cuh"

using wd_host::OnDevice;
using wd_host::set_error;

namespace {

struct Sequence {
    std::vector<int> pages;
    int length = 0;
};

}  // namespace

// The device's book (wd_kv_layout.cuh) has a mirror here; a call changes the mirror and sends the words that differ.
struct wd_kv_cache {
    wd_kv_config cfg{};
    wd::KvShape shape{};
    std::vector<Sequence> seqs;
    std::vector<int> holders;               // of each page
    std::vector<int> free_pages;            // last one goes first
    std::vector<int> book;
    std::vector<int> changed;               // words to send, each of them once
    std::vector<char> dirty;                // those in `changed`
    std::vector<int2> copies;               // pages to copy: from, to
    int table_at = 0, rows = 0, max_rows = 0, items = 0;        // rows of the step, the most of one sequence's, page items

    int n_sm = 0;
    uint8_t *d_pool = nullptr;
    float *d_scales = nullptr, *d_part = nullptr, *d_cta_part = nullptr;
    int *d_book = nullptr, *d_index = nullptr;
    unsigned *d_arrived = nullptr, *d_status = nullptr;
    int2 *d_reach = nullptr;
    size_t pool_layer = 0, scales_layer = 0;
    const char *last_kernel = "";           // of wd_kv_attend
    bool graphs = false;                    // a call has been captured: replays look for the step and the pages in the device's book
    bool broken = false;                    // a launch failed half-way: mirror and device may differ

    bool host_only() const { return cfg.device < 0; }
    int page_tokens() const { return cfg.page_tokens; }
    int pages_for(int tokens) const { return (tokens + cfg.page_tokens - 1) / cfg.page_tokens; }

    void set(size_t at, int value) {
        if (book[at] == value) return;
        book[at] = value;
        if (dirty[at]) return;
        dirty[at] = 1;
        changed.push_back(static_cast<int>(at));
    }
    void set_page(int seq, int i, int page) { set(table_at + static_cast<size_t>(seq) * shape.max_pages + i, page); }
    int take_page() {
        const int p = free_pages.back();
        free_pages.pop_back();
        holders[p] = 1;
        return p;
    }
    void release(int page) {
        if (--holders[page] == 0) free_pages.push_back(page);
    }
    void cut(Sequence &s, int length) {
        const int keep = pages_for(length);
        while (static_cast<int>(s.pages.size()) > keep) {
            release(s.pages.back());
            s.pages.pop_back();
        }
        s.length = length;
    }
    void end_step() {
        set(0, 0);
        set(1, 0);
        set(2, 0);
        rows = max_rows = items = 0;
    }
};

namespace {

int check_seq(const wd_kv_cache *c, int seq) {
    if (seq < 0 || seq >= c->cfg.max_seqs)
        return set_error(WD_E_INVALID, "key/value cache: sequence " + std::to_string(seq) + " of " + std::to_string(c->cfg.max_seqs));
    return WD_OK;
}

int rows_type(int type, int *out) {
    if (type == WD_TYPE_F32) *out = wd::kRowsF32;
    else if (type == WD_TYPE_F16) *out = wd::kRowsF16;
    else if (type == WD_TYPE_BF16) *out = wd::kRowsBF16;
    else return set_error(WD_E_INVALID, "key/value cache: rows are F32, F16 or BF16");
    return WD_OK;
}
size_t rows_size(int type) { return type == wd::kRowsF32 ? 4 : 2; }

int check_rows(const void *p, size_t size, long long *stride, long long least, const char *what) {
    if (!p) return set_error(WD_E_INVALID, std::string("key/value cache: ") + what + " is null");
    if (reinterpret_cast<uintptr_t>(p) % size) return set_error(WD_E_INVALID, std::string("key/value cache: ") + what + " is not aligned to its type");
    if (*stride == 0) *stride = least;
    if (*stride < least) return set_error(WD_E_INVALID, std::string("key/value cache: rows of ") + what + " overlap");
    return WD_OK;
}

// Calls that change the book on the host may not be part of a graph: a replay would repeat the change of the first time.
int check_not_captured(const wd_kv_cache *c, cudaStream_t s) {
    if (c->broken) return set_error(WD_E_STATE, "key/value cache: an earlier call failed on the device");
    if (c->host_only()) return WD_OK;
    cudaGetLastError();         // what an earlier call failed with was said then
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    const cudaError_t ce = cudaStreamIsCapturing(s, &st);
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return set_error(WD_E_STATE, std::string("key/value cache: ") + cudaGetErrorString(ce));
    }
    if (st != cudaStreamCaptureStatusNone) return set_error(WD_E_STATE, "key/value cache: sequences cannot be changed, nor a step without rows taken, while a graph is captured");
    return WD_OK;
}
int check_device(const wd_kv_cache *c) {
    if (!c) return set_error(WD_E_INVALID, "key/value cache: null handle");
    if (c->host_only()) return set_error(WD_E_STATE, "key/value cache: created without a device");
    if (c->broken) return set_error(WD_E_STATE, "key/value cache: an earlier call failed on the device");
    cudaGetLastError();
    return WD_OK;
}

int flush(wd_kv_cache *c, cudaStream_t s);
// Changes that no kernel reads before the next begin, read or keep wait for it (pages change hands only there), unless replays of captured calls may come before:
// they look for the step and for the sequences' pages in the device's book.
int later(wd_kv_cache *c, cudaStream_t s) {
    if (c->host_only()) {
        for (int at : c->changed) c->dirty[at] = 0;
        c->changed.clear();
        return WD_OK;
    }
    if (!c->graphs) return WD_OK;
    OnDevice on(c->cfg.device);
    return flush(c, s);
}
// Whether the call becomes part of a graph; then changes do not wait.
int note_capture(wd_kv_cache *c, cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    WD_TRY_CUDA(cudaStreamIsCapturing(s, &st));
    if (st != cudaStreamCaptureStatusNone) c->graphs = true;
    return WD_OK;
}

template <int N>
void send_words(wd_kv_cache *c, size_t from, cudaStream_t s) {
    wd::KvWords<N> w;
    w.n = static_cast<int>(std::min<size_t>(N, c->changed.size() - from));
    for (int i = 0; i < w.n; ++i) {
        const int at = c->changed[from + i];
        w.w[i] = make_int2(at, c->book[at]);
        c->dirty[at] = 0;
    }
    wd::kv_words_kernel<N><<<1, 256, 0, s>>>(w, c->d_book);
}
// What the call changed goes to the device: pages first, then the words that name them.
int flush(wd_kv_cache *c, cudaStream_t s) {
    if (c->host_only()) {
        c->copies.clear();
        return later(c, s);
    }
    c->broken = true;
    const size_t page_bytes = wd::kv_page_bytes(c->shape);
    for (size_t at = 0; at < c->copies.size(); at += wd::kCopyPairs) {
        wd::KvCopy k;
        k.pool = c->d_pool;
        k.scales = c->d_scales;
        k.pool_layer = c->pool_layer;
        k.scales_layer = c->scales_layer;
        k.page_bytes = page_bytes;
        k.page_scales = c->cfg.n_kv_heads * 2;
        const size_t n = std::min<size_t>(wd::kCopyPairs, c->copies.size() - at);
        std::memcpy(k.pair, c->copies.data() + at, n * sizeof(int2));
        const unsigned x = static_cast<unsigned>(std::min<size_t>(64, (page_bytes / 16 + 1023) / 1024));
        wd::kv_copy_kernel<<<dim3(x, static_cast<unsigned>(n), c->cfg.n_layers), 256, 0, s>>>(k);
    }
    c->copies.clear();
    for (size_t at = 0; at < c->changed.size();) {
        const size_t left = c->changed.size() - at;
        if (left <= 60) send_words<60>(c, at, s), at += 60;
        else if (left <= 500) send_words<500>(c, at, s), at += 500;
        else send_words<4000>(c, at, s), at += 4000;
    }
    c->changed.clear();
    WD_TRY_CUDA(cudaGetLastError());
    c->broken = false;
    return WD_OK;
}

template <class F>
int by_codes(const wd_kv_cache *c, F &&f) {
    return c->shape.e4m3 ? f(std::true_type{}) : f(std::false_type{});
}

template <class F>
int by_rows_and_codes(const wd_kv_cache *c, int rows, F &&f) {
    return by_codes(c, [&](auto e4m3) {
        return rows == wd::kRowsF32 ? f(0.0f, e4m3) : rows == wd::kRowsF16 ? f(__half(), e4m3) : f(__nv_bfloat16(), e4m3);
    });
}

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
Choice choose(const wd_kv_cache *c, bool f32, int window) {
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

}  // namespace

extern "C" {

int wd_kv_create(const wd_kv_config *cfg, wd_kv_cache **out) {
    return wd_host::guarded([&]() -> int {
        if (!cfg || !out) return set_error(WD_E_INVALID, "null argument");
        *out = nullptr;
        const wd_kv_config &c = *cfg;
        if (c.n_layers < 1 || c.n_layers > 4096) return set_error(WD_E_INVALID, "key/value cache: n_layers must be 1 to 4096");
        if (c.n_kv_heads < 1 || c.n_heads < 1 || c.n_heads % c.n_kv_heads || c.n_heads > 4096)
            return set_error(WD_E_INVALID, "key/value cache: n_heads must be a multiple of n_kv_heads, at most 4096");
        if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 96 && c.head_dim != 128 && c.head_dim != 256)
            return set_error(WD_E_INVALID, "key/value cache: head_dim must be 32, 64, 96, 128 or 256");
        if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
            return set_error(WD_E_INVALID, "key/value cache: page_tokens must be 16, 32, 64 or 128");
        if (c.codes != WD_KV_INT8 && c.codes != WD_KV_E4M3) return set_error(WD_E_INVALID, "key/value cache: codes must be WD_KV_INT8 or WD_KV_E4M3");
        if (c.n_pages < 1 || c.max_seqs < 1 || c.max_seqs > wd::kAttMaxSeqs) return set_error(WD_E_INVALID, "key/value cache: n_pages >= 1 and max_seqs 1 to 1024 are wanted");
        if (c.max_context < 1 || c.max_context > (1 << 24)) return set_error(WD_E_INVALID, "key/value cache: max_context must be 1 to 2^24");
        if (c.device < -1) return set_error(WD_E_INVALID, "key/value cache: device");
        std::unique_ptr<wd_kv_cache, void (*)(wd_kv_cache *)> k(new wd_kv_cache, wd_kv_destroy);
        k->cfg = c;
        k->shape = wd::KvShape{c.n_heads, c.n_kv_heads, c.head_dim, c.page_tokens == 16 ? 4 : c.page_tokens == 32 ? 5 : c.page_tokens == 64 ? 6 : 7,
                               c.codes == WD_KV_E4M3, k->pages_for(c.max_context)};
        k->table_at = wd::kKvHead + c.max_seqs * wd::kKvStepWords;
        const size_t words = k->table_at + static_cast<size_t>(c.max_seqs) * k->shape.max_pages;
        if (words > INT_MAX / 2) return set_error(WD_E_INVALID, "key/value cache: max_seqs times max_context is too large for one table");
        // (more than any device has, and more than 64 bits count; where there is less, the device says so)
        if (static_cast<double>(wd::kv_page_bytes(k->shape)) * c.n_pages * c.n_layers > 0x1p42) return set_error(WD_E_NOMEM, "key/value cache: more than 4 TiB of pages do not fit");
        k->book.assign(words, 0);
        k->dirty.assign(words, 0);
        k->seqs.resize(c.max_seqs);
        k->holders.assign(c.n_pages, 0);
        k->free_pages.resize(c.n_pages);
        for (int i = 0; i < c.n_pages; ++i) k->free_pages[i] = c.n_pages - 1 - i;
        k->pool_layer = static_cast<size_t>(c.n_pages) * wd::kv_page_bytes(k->shape);
        k->scales_layer = static_cast<size_t>(c.n_pages) * c.n_kv_heads * 2;
        if (k->host_only()) {
            *out = k.release();
            return WD_OK;
        }
        OnDevice on(c.device);
        if (!on.ok()) return set_error(WD_E_INVALID, "key/value cache: no device " + std::to_string(c.device));
        WD_TRY_CUDA(cudaDeviceGetAttribute(&k->n_sm, cudaDevAttrMultiProcessorCount, c.device));
        auto alloc = [&](auto **p, size_t bytes) {
            const cudaError_t ce = cudaMalloc(reinterpret_cast<void **>(p), bytes);
            if (ce == cudaSuccess) return cudaMemsetAsync(*p, 0, bytes, cudaStreamLegacy);
            cudaGetLastError();
            return ce;
        };
        const size_t part = static_cast<size_t>(k->n_sm) * 2 * wd::kAttMaxRows * (c.head_dim + 4) * 4;     // of a CTA, or of a worker
        // (zeros are codes, so that no part of a page ever holds what is not one)
        if (alloc(&k->d_pool, k->pool_layer * c.n_layers) != cudaSuccess || alloc(&k->d_scales, k->scales_layer * c.n_layers * 4) != cudaSuccess ||
            alloc(&k->d_part, part * wd::kAttWorkers) != cudaSuccess || alloc(&k->d_cta_part, part) != cudaSuccess || alloc(&k->d_book, words * 4) != cudaSuccess ||
            alloc(&k->d_index, (static_cast<size_t>(c.max_context) + k->shape.max_pages) * 4) != cudaSuccess ||
            alloc(&k->d_arrived, static_cast<size_t>(k->n_sm) * 4) != cudaSuccess || alloc(&k->d_status, 16) != cudaSuccess ||
            alloc(&k->d_reach, static_cast<size_t>(c.n_layers) * c.n_kv_heads * sizeof(int2)) != cudaSuccess)
            return set_error(WD_E_NOMEM, "key/value cache: " + std::to_string((k->pool_layer * c.n_layers) >> 20) + " MiB of pages do not fit");
        WD_TRY_CUDA(cudaStreamSynchronize(cudaStreamLegacy));
        *out = k.release();
        return WD_OK;
    });
}

void wd_kv_destroy(wd_kv_cache *c) {
    if (!c) return;
    if (!c->host_only()) {
        OnDevice on(c->cfg.device);
        for (void *p : {static_cast<void *>(c->d_pool), static_cast<void *>(c->d_scales), static_cast<void *>(c->d_part), static_cast<void *>(c->d_cta_part), static_cast<void *>(c->d_book),
                        static_cast<void *>(c->d_index), static_cast<void *>(c->d_arrived), static_cast<void *>(c->d_status), static_cast<void *>(c->d_reach)})
            if (p) cudaFree(p);
    }
    delete c;
}

int wd_kv_begin(wd_kv_cache *c, int n, const int *seqs, const int *counts, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (!c || n < 0 || (n > 0 && (!seqs || !counts))) return set_error(WD_E_INVALID, "null argument");
        if (n > c->cfg.max_seqs) return set_error(WD_E_INVALID, "key/value cache: a step of more sequences than there are");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        std::vector<char> named(c->cfg.max_seqs, 0);
        std::unordered_map<int, int> left;          // holders of a page as the copies in front leave them
        long long rows = 0, need = 0;
        for (int i = 0; i < n; ++i) {
            if (int rc = check_seq(c, seqs[i])) return rc;
            if (named[seqs[i]]++) return set_error(WD_E_INVALID, "key/value cache: a step names sequence " + std::to_string(seqs[i]) + " twice");
            const Sequence &q = c->seqs[seqs[i]];
            if (counts[i] < 0 || counts[i] > c->cfg.max_context - q.length)
                return set_error(WD_E_INVALID, "key/value cache: " + std::to_string(counts[i]) + " tokens behind " + std::to_string(q.length) + " of at most " +
                                                   std::to_string(c->cfg.max_context));
            rows += counts[i];
            need += c->pages_for(q.length + counts[i]) - static_cast<int>(q.pages.size());
            if (counts[i] > 0 && q.length % c->page_tokens()) {
                auto at = left.emplace(q.pages.back(), c->holders[q.pages.back()]).first;
                if (at->second > 1) --at->second, ++need;
            }
        }
        if (rows * c->cfg.n_heads > INT_MAX / 2) return set_error(WD_E_INVALID, "key/value cache: too many rows in a step");        // (kernels count rows of heads in 32 bits)
        if (need > static_cast<long long>(c->free_pages.size()))
            return set_error(WD_E_NOMEM, "key/value cache: " + std::to_string(need) + " pages wanted, " + std::to_string(c->free_pages.size()) + " free");
        if (int rc = check_not_captured(c, s)) return rc;
        // (no memory is asked for between the first change and the last)
        c->changed.reserve(c->changed.size() + static_cast<size_t>(n) * 5 + need + 8);
        c->copies.reserve(n);
        for (int i = 0; i < n; ++i) c->seqs[seqs[i]].pages.reserve(c->pages_for(c->seqs[seqs[i]].length + counts[i]));
        c->rows = c->max_rows = c->items = 0;
        for (int i = 0; i < n; ++i) {
            Sequence &q = c->seqs[seqs[i]];
            const int begin = q.length, end = begin + counts[i];
            if (counts[i] > 0 && begin % c->page_tokens() && c->holders[q.pages.back()] > 1) {
                const int old = q.pages.back(), fresh = c->take_page();
                c->release(old);
                q.pages.back() = fresh;
                c->set_page(seqs[i], static_cast<int>(q.pages.size()) - 1, fresh);
                c->copies.push_back(make_int2(old, fresh));
            }
            while (static_cast<int>(q.pages.size()) < c->pages_for(end)) {
                q.pages.push_back(c->take_page());
                c->set_page(seqs[i], static_cast<int>(q.pages.size()) - 1, q.pages.back());
            }
            q.length = end;
            const size_t e = wd::kKvHead + static_cast<size_t>(i) * wd::kKvStepWords;
            c->set(e, seqs[i]);
            c->set(e + 1, c->rows);
            c->set(e + 2, counts[i]);
            c->set(e + 3, end);
            c->set(e + 4, c->items);
            c->rows += counts[i];
            c->max_rows = std::max(c->max_rows, counts[i]);
            if (counts[i] > 0) c->items += (end - 1) / c->page_tokens() - begin / c->page_tokens() + 1;
        }
        c->set(0, n);
        c->set(1, c->rows);
        c->set(2, c->items);
        OnDevice on(c->host_only() ? 0 : c->cfg.device);
        return flush(c, s);
    });
}

int wd_kv_append(wd_kv_cache *c, int layer, const void *k_dev, const void *v_dev, int type, int64_t k_stride, int64_t v_stride, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (int rc = check_device(c)) return rc;
        if (layer < 0 || layer >= c->cfg.n_layers) return set_error(WD_E_INVALID, "key/value cache: layer out of range");
        wd::KvAppend p;
        int rows_of = 0;
        if (int rc = rows_type(type, &rows_of)) return rc;
        if (c->book[0] == 0) return set_error(WD_E_STATE, "key/value cache: no step has begun");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c->items == 0) return check_not_captured(c, s);         // (no rows: nothing is asked of their address, and a graph would hold nothing)
        const size_t size = rows_size(rows_of);
        p.stride[0] = k_stride;
        p.stride[1] = v_stride;
        const long long width = static_cast<long long>(c->cfg.n_kv_heads) * c->cfg.head_dim;
        if (int rc = check_rows(k_dev, size, &p.stride[0], width, "k")) return rc;
        if (int rc = check_rows(v_dev, size, &p.stride[1], width, "v")) return rc;
        OnDevice on(c->cfg.device);
        if (int rc = note_capture(c, s)) return rc;
        p.pool = c->d_pool + layer * c->pool_layer;
        p.scales = c->d_scales + layer * c->scales_layer;
        p.reach = c->d_reach + static_cast<size_t>(layer) * c->cfg.n_kv_heads;
        p.book = c->d_book;
        p.table = c->d_book + c->table_at;
        p.rows[0] = k_dev;
        p.rows[1] = v_dev;
        p.status = c->d_status;
        p.s = c->shape;
        for (int i = 0; i < 2; ++i) p.vec[i] = reinterpret_cast<uintptr_t>(p.rows[i]) % 16 == 0 && p.stride[i] * size % 16 == 0;
        const dim3 grid(static_cast<unsigned>(c->items), c->cfg.n_kv_heads, 2);
        const size_t smem = static_cast<size_t>(c->cfg.page_tokens) * c->cfg.head_dim;
        // few tokens a page: a warp reads them at once, and more threads would only meet at the barriers
        const bool small = static_cast<long long>(std::min(c->max_rows, c->cfg.page_tokens)) * c->cfg.head_dim <= 2048;
        return by_rows_and_codes(c, rows_of, [&](auto t, auto e4m3) {
            using T = decltype(t);
            if (small) wd::kv_append_kernel<T, decltype(e4m3)::value, 64><<<grid, 64, smem, s>>>(p);
            else wd::kv_append_kernel<T, decltype(e4m3)::value, 256><<<grid, 256, smem, s>>>(p);
            WD_TRY_CUDA(cudaGetLastError());
            return WD_OK;
        });
    });
}

int wd_kv_attend(wd_kv_cache *c, int layer, const void *q_dev, void *out_dev, int type, float scale, int window, int64_t q_stride, int64_t out_stride, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (int rc = check_device(c)) return rc;
        if (layer < 0 || layer >= c->cfg.n_layers) return set_error(WD_E_INVALID, "key/value cache: layer out of range");
        if (!(scale > 0.0f && scale * 1.4426950408889634 <= 3.4028234663852886e38)) return set_error(WD_E_INVALID, "key/value cache: the scale of the scores must be positive and finite");
        if (window < 0) return set_error(WD_E_INVALID, "key/value cache: a window is 0 (none) or at least 1");
        wd::KvAttend p;
        if (int rc = rows_type(type, &p.type)) return rc;
        if (c->book[0] == 0) return set_error(WD_E_STATE, "key/value cache: no step has begun");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (c->rows == 0) return check_not_captured(c, s);
        if (window >= c->cfg.max_context) window = 0;
        p.q_stride = q_stride;
        p.out_stride = out_stride;
        const long long width = static_cast<long long>(c->cfg.n_heads) * c->cfg.head_dim;
        if (int rc = check_rows(q_dev, rows_size(p.type), &p.q_stride, width, "q")) return rc;
        if (int rc = check_rows(out_dev, rows_size(p.type), &p.out_stride, width, "out")) return rc;
        if (q_dev == out_dev && p.q_stride != p.out_stride) return set_error(WD_E_INVALID, "key/value cache: out over q needs q's stride");
        OnDevice on(c->cfg.device);
        if (int rc = note_capture(c, s)) return rc;
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
        p.window = window;
        p.max_seqs = c->cfg.max_seqs;
        p.vec = reinterpret_cast<uintptr_t>(q_dev) % 16 == 0 && p.q_stride * rows_size(p.type) % 16 == 0;
        p.s = c->shape;
        const long long group = static_cast<long long>(c->max_rows) * (c->cfg.n_heads / c->cfg.n_kv_heads);
        const Choice by = choose(c, p.type == wd::kRowsF32, window);
        c->last_kernel = by.prompt ? by.split ? "kv_prompt_kernel, kv_prompt_join_kernel" : "kv_prompt_kernel" : "kv_attend_kernel";
        if (by.prompt) {
            wd::KvPrompt r;
            r.pool = p.pool, r.scales = p.scales, r.reach = c->d_reach + static_cast<size_t>(layer) * c->cfg.n_kv_heads, r.book = p.book, r.table = p.table, r.q = p.q, r.out = p.out;
            r.q_stride = p.q_stride, r.out_stride = p.out_stride, r.status = p.status, r.scale_log2 = p.scale_log2;
            r.type = p.type, r.window = p.window, r.s = p.s, r.part = c->d_part, r.ctas = c->n_sm;
            r.split = by.split;         // (the kernels count the items of the step that is current when they run)
            const size_t size = rows_size(p.type);
            r.vec = (reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev)) % 16 == 0 && p.q_stride * size % 16 == 0 && p.out_stride * size % 16 == 0;
            switch (c->cfg.head_dim) {
                case 32: return prompt_of<32>(c, r, s);
                case 64: return prompt_of<64>(c, r, s);
                case 96: return prompt_of<96>(c, r, s);
                case 128: return prompt_of<128>(c, r, s);
                default: return prompt_of<256>(c, r, s);
            }
        }
        const bool few = group <= 8;
        switch (c->cfg.head_dim) {
            case 32: return attend_of<32>(c, p, few, s);
            case 64: return attend_of<64>(c, p, few, s);
            case 96: return attend_of<96>(c, p, few, s);
            case 128: return attend_of<128>(c, p, few, s);
            default: return attend_of<256>(c, p, few, s);
        }
    });
}

int wd_kv_read(wd_kv_cache *c, int layer, int n, const int *seqs, const int *firsts, const int *counts, void *k_dev, void *v_dev, int type, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (int rc = check_device(c)) return rc;
        if (layer < -1 || layer >= c->cfg.n_layers) return set_error(WD_E_INVALID, "key/value cache: layer out of range");
        if (n < 0 || (n > 0 && (!seqs || !firsts || !counts)) || (!k_dev && !v_dev)) return set_error(WD_E_INVALID, "null argument");
        wd::KvRead p;
        int rows_of = 0;
        if (int rc = rows_type(type, &rows_of)) return rc;
        const size_t size = rows_size(rows_of);
        for (const void *o : {k_dev, v_dev})
            if (reinterpret_cast<uintptr_t>(o) % size) return set_error(WD_E_INVALID, "key/value cache: an output is not aligned to its type");
        long long rows = 0;
        for (int i = 0; i < n; ++i) {
            if (int rc = check_seq(c, seqs[i])) return rc;
            const int length = c->seqs[seqs[i]].length;
            if (firsts[i] < 0 || counts[i] < 0 || firsts[i] > length || counts[i] > length - firsts[i])
                return set_error(WD_E_INVALID, "key/value cache: tokens " + std::to_string(firsts[i]) + " to " + std::to_string(static_cast<long long>(firsts[i]) + counts[i]) +
                                                   " of a sequence of " + std::to_string(length));
            rows += counts[i];
        }
        if (rows > INT_MAX / 2) return set_error(WD_E_INVALID, "key/value cache: too many rows in a read");
        if (rows == 0) return WD_OK;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (!c->changed.empty())
            if (int rc = check_not_captured(c, s)) return rc;
        OnDevice on(c->cfg.device);
        if (int rc = note_capture(c, s)) return rc;
        if (int rc = flush(c, s)) return rc;
        const size_t width = static_cast<size_t>(c->cfg.n_kv_heads) * c->cfg.head_dim;
        const int layers = layer < 0 ? c->cfg.n_layers : 1;
        p.pool = c->d_pool + (layer < 0 ? 0 : layer) * c->pool_layer;
        p.scales = c->d_scales + (layer < 0 ? 0 : layer) * c->scales_layer;
        p.table = c->d_book + c->table_at;
        p.out[0] = k_dev;
        p.out[1] = v_dev;
        p.pool_layer = c->pool_layer;
        p.scales_layer = c->scales_layer;
        p.out_layer = static_cast<size_t>(rows) * width;
        p.vec = (reinterpret_cast<uintptr_t>(k_dev) | reinterpret_cast<uintptr_t>(v_dev)) % 16 == 0;       // (a row is a multiple of 64 bytes)
        p.s = c->shape;
        int row = 0;
        for (int i = 0; i < n;) {
            int items = 0;
            p.n = 0;
            for (; i < n && p.n < wd::kReadEntries; ++i) {
                if (counts[i] == 0) continue;
                p.e[p.n++] = wd::KvReadEntry{seqs[i], firsts[i], counts[i], row, items};
                items += (firsts[i] + counts[i] - 1) / wd::kKvSub - firsts[i] / wd::kKvSub + 1;
                row += counts[i];
            }
            if (p.n == 0) continue;
            const dim3 grid(static_cast<unsigned>(items), static_cast<unsigned>(layers));
            const int rc = by_rows_and_codes(c, rows_of, [&](auto t, auto e4m3) {
                wd::kv_read_kernel<decltype(t), decltype(e4m3)::value><<<grid, wd::kReadThreads, 0, s>>>(p);
                WD_TRY_CUDA(cudaGetLastError());
                return WD_OK;
            });
            if (rc) return rc;
        }
        return WD_OK;
    });
}

int wd_kv_fork(wd_kv_cache *c, int src, int n, const int *dsts, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (!c || n < 0 || (n > 0 && !dsts)) return set_error(WD_E_INVALID, "null argument");
        if (int rc = check_seq(c, src)) return rc;
        std::vector<char> named(c->cfg.max_seqs, 0);
        for (int i = 0; i < n; ++i) {
            if (int rc = check_seq(c, dsts[i])) return rc;
            if (dsts[i] == src || named[dsts[i]]++) return set_error(WD_E_INVALID, "key/value cache: a fork goes to other sequences, to each of them once");
            if (c->seqs[dsts[i]].length > 0) return set_error(WD_E_STATE, "key/value cache: sequence " + std::to_string(dsts[i]) + " is not free");
        }
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (int rc = check_not_captured(c, s)) return rc;
        const Sequence &from = c->seqs[src];
        c->changed.reserve(c->changed.size() + from.pages.size() * n);
        for (int i = 0; i < n; ++i) c->seqs[dsts[i]].pages.reserve(from.pages.size());
        for (int i = 0; i < n; ++i) {
            c->seqs[dsts[i]] = from;
            for (size_t j = 0; j < from.pages.size(); ++j) {
                ++c->holders[from.pages[j]];
                c->set_page(dsts[i], static_cast<int>(j), from.pages[j]);
            }
        }
        return later(c, s);
    });
}

int wd_kv_truncate(wd_kv_cache *c, int seq, int length, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (!c) return set_error(WD_E_INVALID, "null argument");
        if (int rc = check_seq(c, seq)) return rc;
        if (length < 0 || length > c->seqs[seq].length) return set_error(WD_E_INVALID, "key/value cache: a sequence can be cut to 0 up to its length");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (int rc = check_not_captured(c, s)) return rc;
        c->changed.reserve(c->changed.size() + 3);
        c->cut(c->seqs[seq], length);
        c->end_step();
        return later(c, s);
    });
}

int wd_kv_free(wd_kv_cache *c, int n, const int *seqs, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (!c || n < 0 || (n > 0 && !seqs)) return set_error(WD_E_INVALID, "null argument");
        for (int i = 0; i < n; ++i)
            if (int rc = check_seq(c, seqs[i])) return rc;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (int rc = check_not_captured(c, s)) return rc;
        c->changed.reserve(c->changed.size() + 3);
        for (int i = 0; i < n; ++i) c->cut(c->seqs[seqs[i]], 0);
        c->end_step();
        return later(c, s);
    });
}

int wd_kv_keep(wd_kv_cache *c, int seq, int first, int n, const int *index, void *stream) {
    return wd_host::guarded([&]() -> int {
        if (!c || n < 0 || (n > 0 && !index)) return set_error(WD_E_INVALID, "null argument");
        if (int rc = check_seq(c, seq)) return rc;
        Sequence &q = c->seqs[seq];
        if (first < 0 || first > q.length) return set_error(WD_E_INVALID, "key/value cache: keep begins behind the sequence's end");
        for (int i = 0; i < n; ++i)
            if (index[i] < 0 || index[i] >= q.length - first || (i > 0 && index[i] <= index[i - 1]))
                return set_error(WD_E_INVALID, "key/value cache: kept tokens go up, from 0 to the sequence's last token behind `first`");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (int rc = check_not_captured(c, s)) return rc;
        int still = 0;          // tokens that stay where they are
        while (still < n && index[still] == still) ++still;
        const int from = first + still, kept = n - still, end = first + n;
        if (kept == 0) {
            c->changed.reserve(c->changed.size() + 3);
            c->cut(q, end);
            c->end_step();
            return later(c, s);
        }
        const int page0 = from / c->page_tokens(), pages = c->pages_for(end) - page0;
        // Into new pages, all at once, where there are enough of them; else in place, page by page, but never into a page that others hold.
        const bool fresh = static_cast<int>(c->free_pages.size()) >= pages;
        int shared = 0;
        for (int i = 0; i < pages; ++i) shared += c->holders[q.pages[page0 + i]] > 1;
        if (!fresh && shared > static_cast<int>(c->free_pages.size()))
            return set_error(WD_E_NOMEM, "key/value cache: " + std::to_string(shared) + " pages wanted, " + std::to_string(c->free_pages.size()) + " free");
        std::vector<int> words(index + still, index + n), to(pages);
        words.reserve(words.size() + pages);
        c->changed.reserve(c->changed.size() + pages + 3);
        c->free_pages.reserve(c->free_pages.size() + q.pages.size());
        for (int &w : words) w -= still;
        for (int i = 0; i < pages; ++i) to[i] = fresh || c->holders[q.pages[page0 + i]] > 1 ? c->take_page() : q.pages[page0 + i];
        OnDevice on(c->host_only() ? 0 : c->cfg.device);
        if (!c->host_only()) {
            if (int rc = flush(c, s)) return rc;        // the table as it was
            c->broken = true;
            words.insert(words.end(), to.begin(), to.end());
            for (size_t at = 0; at < words.size();) {
                const int left = static_cast<int>(words.size() - at);
                auto send = [&](auto &r, int most) {
                    r.n = std::min(left, most);
                    r.offset = static_cast<int>(at);
                    std::memcpy(r.w, words.data() + at, static_cast<size_t>(r.n) * 4);
                    at += r.n;
                };
                if (left <= 900) {
                    wd::KvRun<900> r;
                    send(r, 900);
                    wd::kv_run_kernel<900><<<1, 256, 0, s>>>(r, c->d_index);
                } else {
                    wd::KvRun<8000> r;
                    send(r, 8000);
                    wd::kv_run_kernel<8000><<<1, 256, 0, s>>>(r, c->d_index);
                }
            }
            wd::KvKeep p;
            p.pool = c->d_pool;
            p.scales = c->d_scales;
            p.table = c->d_book + c->table_at + static_cast<size_t>(seq) * c->shape.max_pages;
            p.index = c->d_index;
            p.to = c->d_index + kept;
            p.pool_layer = c->pool_layer;
            p.scales_layer = c->scales_layer;
            p.first = from;
            p.kept = kept;
            p.page0 = page0;
            p.pages = pages;
            p.s = c->shape;
            const size_t smem = static_cast<size_t>(c->cfg.page_tokens) * c->cfg.head_dim;
            if (fresh) {
                const dim3 grid(pages, c->cfg.n_layers, (c->cfg.n_kv_heads + wd::kKeepHeads - 1) / wd::kKeepHeads);
                if (c->shape.e4m3) wd::kv_keep_new_kernel<true><<<grid, wd::kKeepThreads, 0, s>>>(p);
                else wd::kv_keep_new_kernel<false><<<grid, wd::kKeepThreads, 0, s>>>(p);
            } else {
                const int per = std::max(1, 65535 / c->cfg.n_kv_heads);         // (the second index of a grid ends at 65,535)
                for (int l = 0; l < c->cfg.n_layers; l += per) {
                    const dim3 grid(1, static_cast<unsigned>(std::min(per, c->cfg.n_layers - l) * c->cfg.n_kv_heads), 2);
                    wd::KvKeep pl = p;
                    pl.pool += l * c->pool_layer;
                    pl.scales += l * c->scales_layer;
                    if (c->shape.e4m3) wd::kv_keep_kernel<true><<<grid, wd::kKeepThreads, smem, s>>>(pl);
                    else wd::kv_keep_kernel<false><<<grid, wd::kKeepThreads, smem, s>>>(pl);
                }
            }
            WD_TRY_CUDA(cudaGetLastError());
            c->broken = false;
        }
        for (int i = 0; i < pages; ++i) {
            if (to[i] == q.pages[page0 + i]) continue;
            c->release(q.pages[page0 + i]);
            q.pages[page0 + i] = to[i];
            c->set_page(seq, page0 + i, to[i]);
        }
        c->cut(q, end);
        c->end_step();
        return c->host_only() ? later(c, s) : flush(c, s);
    });
}

int wd_kv_length(const wd_kv_cache *c, int seq) {
    if (!c) return set_error(WD_E_INVALID, "null argument");
    if (int rc = check_seq(c, seq)) return rc;
    return c->seqs[seq].length;
}
int wd_kv_free_pages(const wd_kv_cache *c) { return c ? static_cast<int>(c->free_pages.size()) : set_error(WD_E_INVALID, "null argument"); }
int wd_kv_pages(const wd_kv_cache *c, int seq, int *pages, int cap) {
    if (!c || cap < 0 || (cap > 0 && !pages)) return set_error(WD_E_INVALID, "null argument");
    if (int rc = check_seq(c, seq)) return rc;
    const std::vector<int> &p = c->seqs[seq].pages;
    std::copy_n(p.begin(), std::min<size_t>(p.size(), cap), pages);
    return static_cast<int>(p.size());
}
const char *wd_kv_kernel_name(const wd_kv_cache *c) { return c ? c->last_kernel : ""; }
int wd_kv_status(wd_kv_cache *c, int *status) {
    return wd_host::guarded([&]() -> int {
        if (int rc = check_device(c)) return rc;
        if (!status) return set_error(WD_E_INVALID, "null argument");
        OnDevice on(c->cfg.device);
        WD_TRY_CUDA(cudaDeviceSynchronize());
        unsigned st = 0;
        WD_TRY_CUDA(cudaMemcpy(&st, c->d_status, 4, cudaMemcpyDeviceToHost));
        WD_TRY_CUDA(cudaMemset(c->d_status, 0, 16));
        *status = static_cast<int>(st);
        if (st & (wd::kErrCopyTimeout | wd::kErrBarrierTimeout)) {
            WD_TRY_CUDA(cudaMemset(c->d_arrived, 0, static_cast<size_t>(c->n_sm) * 4));
            WD_TRY_CUDA(cudaDeviceSynchronize());
            return set_error(WD_E_DEVICE, "key/value cache: a wait on the device ran out");
        }
        WD_TRY_CUDA(cudaDeviceSynchronize());
        return WD_OK;
    });
}

}  // extern "C"
