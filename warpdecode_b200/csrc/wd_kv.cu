// Host side of the 8-bit key/value cache (wd_kv_*): which sequence holds which pages, the step, and the launches.
#include <climits>
#include <cmath>
#include <cstring>
#include <memory>
#include <unordered_map>

#include "wd_kv_append.cuh"
#include "wd_kv_kernels.cuh"
#include "wd_kv_launch.cuh"

using namespace wd_kv;

namespace {

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
            alloc(&k->d_part, part * wd::kAttWorkers * wd::kTreeUnits / 2) != cudaSuccess || alloc(&k->d_cta_part, part) != cudaSuccess || alloc(&k->d_book, words * 4) != cudaSuccess ||
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
        fill_append(c, layer, k_dev, v_dev, size, &p);
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
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        wd::KvAttend p;
        int rc = WD_OK;
        if (!attend_ready(c, layer, q_dev, out_dev, type, scale, window, q_stride, out_stride, s, p, rc)) return rc;
        OnDevice on(c->cfg.device);
        if (int r = note_capture(c, s)) return r;
        const Choice by = choose(c, p.type == wd::kRowsF32, p.window);
        if (!by.prompt) return attend_few(c, p, s);
        c->last_kernel = by.split ? "kv_prompt_kernel, kv_prompt_join_kernel" : "kv_prompt_kernel";
        wd::KvPrompt r;
        fill_prompt(c, layer, p, by.split, &r);
        switch (c->cfg.head_dim) {
            case 32: return prompt_of<32>(c, r, s);
            case 64: return prompt_of<64>(c, r, s);
            case 96: return prompt_of<96>(c, r, s);
            case 128: return prompt_of<128>(c, r, s);
            default: return prompt_of<256>(c, r, s);
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
