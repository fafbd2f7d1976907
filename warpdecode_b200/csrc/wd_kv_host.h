// What the entry points of the 8-bit key/value cache (wd_kv_*) share on the host: the cache itself, checks of arguments, types of rows and codes.
#pragma once

#include <algorithm>
#include <string>
#include <type_traits>
#include <vector>

#include "wd_host.h"
#include "wd_kv_append.cuh"

// The device's book (wd_kv_layout.cuh) has a mirror here; a call changes the mirror and sends the words that differ.
struct wd_kv_cache {
    struct Sequence {
        std::vector<int> pages;
        int length = 0;
    };

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

namespace wd_kv {

using wd_host::OnDevice;
using wd_host::set_error;
using Sequence = wd_kv_cache::Sequence;

inline int check_seq(const wd_kv_cache *c, int seq) {
    if (seq < 0 || seq >= c->cfg.max_seqs)
        return set_error(WD_E_INVALID, "key/value cache: sequence " + std::to_string(seq) + " of " + std::to_string(c->cfg.max_seqs));
    return WD_OK;
}

inline int rows_type(int type, int *out) {
    if (type == WD_TYPE_F32) *out = wd::kRowsF32;
    else if (type == WD_TYPE_F16) *out = wd::kRowsF16;
    else if (type == WD_TYPE_BF16) *out = wd::kRowsBF16;
    else return set_error(WD_E_INVALID, "key/value cache: rows are F32, F16 or BF16");
    return WD_OK;
}
inline size_t rows_size(int type) { return type == wd::kRowsF32 ? 4 : 2; }

inline int check_rows(const void *p, size_t size, long long *stride, long long least, const char *what) {
    if (!p) return set_error(WD_E_INVALID, std::string("key/value cache: ") + what + " is null");
    if (reinterpret_cast<uintptr_t>(p) % size) return set_error(WD_E_INVALID, std::string("key/value cache: ") + what + " is not aligned to its type");
    if (*stride == 0) *stride = least;
    if (*stride < least) return set_error(WD_E_INVALID, std::string("key/value cache: rows of ") + what + " overlap");
    return WD_OK;
}

// Calls that change the book on the host may not be part of a graph: a replay would repeat the change of the first time.
inline int check_not_captured(const wd_kv_cache *c, cudaStream_t s) {
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
inline int check_device(const wd_kv_cache *c) {
    if (!c) return set_error(WD_E_INVALID, "key/value cache: null handle");
    if (c->host_only()) return set_error(WD_E_STATE, "key/value cache: created without a device");
    if (c->broken) return set_error(WD_E_STATE, "key/value cache: an earlier call failed on the device");
    cudaGetLastError();
    return WD_OK;
}
// Whether the call becomes part of a graph; then changes do not wait.
inline int note_capture(wd_kv_cache *c, cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    WD_TRY_CUDA(cudaStreamIsCapturing(s, &st));
    if (st != cudaStreamCaptureStatusNone) c->graphs = true;
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

// A launch that appends to a layer, but for the strides.
inline void fill_append(const wd_kv_cache *c, int layer, const void *k_dev, const void *v_dev, size_t size, wd::KvAppend *p) {
    p->pool = c->d_pool + layer * c->pool_layer;
    p->scales = c->d_scales + layer * c->scales_layer;
    p->reach = c->d_reach + static_cast<size_t>(layer) * c->cfg.n_kv_heads;
    p->book = c->d_book;
    p->table = c->d_book + c->table_at;
    p->rows[0] = k_dev;
    p->rows[1] = v_dev;
    p->status = c->d_status;
    p->s = c->shape;
    for (int i = 0; i < 2; ++i) p->vec[i] = reinterpret_cast<uintptr_t>(p->rows[i]) % 16 == 0 && p->stride[i] * size % 16 == 0;
}

}  // namespace wd_kv
