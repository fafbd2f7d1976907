// Attention over the 8-bit cache for few rows: the last tokens of each of a step's sequences against everything in front of them.
//
//   out[r] = sum_j p_j cv_j sv_j / sum_j p_j,   p_j = 2^(x_j - m),   x_j = (q[r] . ck_j) (2^e scale log2(e) sk_j)
//
// q is brought to F16 row by row: q = 2^e (hi + lo) with |hi| <= 2^15, lo = 0 unless the rows are F32; codes are exact in F16; sums are F32. (2^15 for the
// row's largest element, so that one that is far smaller is not rounded away at F16's lower end: elements are off by 2^-40 of the largest at most.)
// Weights: m is the running maximum of x_j + log2(sv_j). E_j = 2^(7 + x_j - m) makes the denominator, P_j = E_j (2^6 sv_j) <= 2^13 meets the codes (F16,
// hi + lo for F32 rows); the answer is 2^-6 sum P_j cv_j / sum E_j. So a page whose values are small loses nothing beside one whose values are large
// unless its part of the sum is small, and its tokens' weights are counted whatever their values. Within F32: E_j is at least 2^-79 for the token
// with the largest weight where scales are below 2^86 (2^-114 at the largest F32 has), and at most 2^107.
//
// The 2^13 (it divides out) puts the largest weight near the upper end of F16's range, so that the many small weights behind a heavy token are not lost at
// the lower one: a weight is off by half a step of its terms (2^-11 of itself; 2^-22 of two), and by 2^-38 of the row's largest, where F16 ends. So
// n tokens' answer is off by n 2^-38 of the values' size at most. (With the largest weight at 1 it was n 2^-25: the sum of 131,072 tokens that have
// 10 % of the weight behind one that has the rest was off by 2e-2 of itself.)
//
// Products: keys and values are the A operands (16 tokens, or 16 elements of the head), 8 rows of q the B operand, so that a group of up to 8 query
// heads wastes nothing and the codes are expanded once for all of a warp's rows. The weights come out of the first product with tokens along the
// lanes' g and are needed with tokens along t: one 8 x 8 transposition of F16 pairs (movmatrix) each.
//
// Work: a tile is 64 tokens of one kv head, an item the tiles that 8 N8 rows of a head of a sequence see. All items' tiles are numbered through
// (an item counts a few more than it has, for what it costs to begin and end one), and each worker, a warp, takes an equal run of the numbers, whatever
// the sequences' lengths. A worker has a warp beside it that brings its keys and values into a ring of its own by bulk copies. Nothing is waited for
// between workers until all of a CTA's are done; then the parts of items that several of them hold are put together, and those that several CTAs
// hold by the last CTA to arrive, always in the workers' order.
//
// Bound: memory for long work. 131,089 tokens of 8 heads of 128: 58 us, 4.6 TB/s of codes (the copy rate's floor is 42); 64 sequences of 90 to 8,000
// tokens, 8 heads of 64: 46 us, 3.9 TB/s (28): the rest is the way to the first tile and the joining of parts (DRAM is busy for 56 and 48 % of the
// launch, issue slots 30 and 47 %, the tensor pipe 13 and 11 %). Short work is a chain of latencies: 131 tokens, 4 heads of 64: 9 to 10 us, most of them the launch, entry -> table -> page -> tile, and code that an SM fetches for the first time.
#pragma once

#include <type_traits>

#include "wd_kv_layout.cuh"

namespace wd {

constexpr int kAttWorkers = 8, kAttThreads = 512, kAttMaxSeqs = 1024, kAttMaxRows = 16, kAttMaxSlots = 8, kAttEntries = 64, kAttMaxCtas = 256;
// Registers a thread: the warps that compute take what those that copy give back (128 at launch).
constexpr int kAttRegsMore = 192, kAttRegsLess = 64;
static_assert(256 * kAttRegsMore + 256 * kAttRegsLess <= kAttThreads * 128, "more than the block was launched with: the increase would wait for ever");
constexpr float kAttFloor = -1.0e30f;       // a maximum over nothing (scores are below 2^20)
constexpr int kAttTop = 13, kAttScale = 6;              // exponents: of the largest P_j, of what a value scale is multiplied by (F32's largest scale is below 2^122)
constexpr float kAttUnit = 1.0f / (1 << kAttScale);

struct KvAttend {
    const uint8_t *pool;        // of the layer
    const float *scales;        // of the layer
    const int *book;
    const int *table;
    const void *q;
    void *out;
    long long q_stride, out_stride;
    float *part;                // [workers][kAttMaxRows][D + 4]: sums, then maximum and denominator
    float *cta_part;            // [CTAs][2][kAttMaxRows][D + 4]
    unsigned *arrived;          // [CTAs]
    unsigned *status;
    float scale_log2;
    int type, window, workers, slots, max_seqs, vec;          // vec: rows of q lie on boundaries of 16 bytes
    KvShape s;
};

template <int D>
struct AttendPlan {
    static constexpr int kCw = D % 64 == 0 ? 64 : 32;
    static constexpr int kSlot = 64 * D + 64;           // keys or values of a tile; behind the keys 4 x {key scale, log2 of the value scale, 2^6 times the value scale}
    __host__ __device__ static constexpr int q_bytes(int n8, bool split) { return n8 * 8 * D * 2 * (split ? 2 : 1); }
    __host__ __device__ static constexpr int fixed_bytes(int workers, int n8, bool split) { return workers * q_bytes(n8, split) + (kAttMaxSeqs + 2) * 8; }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {        // on sums of 0
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void att_bar() { asm volatile("bar.sync 1, %0;" ::"n"(kAttWorkers * 32) : "memory"); }
// two floats -> F16 pair, and the pair of what that rounding left over
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t half_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return half_pair(a - f.x, b - f.y);
}

// Bounded wait by a count of polls, inline (a call would keep the compiler from moving registers between the warpgroups): a poll suspends the thread
// for 1.3 us, so that the limit is 1.4 s, or 0.3 ms once another wait has run out. What follows reads what is there and ends.
__device__ __forceinline__ void att_wait(uint64_t *bar, uint32_t parity, unsigned *status) {
#pragma unroll 1
    for (unsigned i = 0; i < kSpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 255u) == 255u && *reinterpret_cast<volatile unsigned *>(status) & kErrCopyTimeout) break;
    }
    atomicOr(status, kErrCopyTimeout);
}

// A run's part of an item.
struct AttSegment {
    int seq, row0, count, length, head, item_row, rows;         // rows: of the item, from item_row on
    int lo, hi;                 // tiles of 64 tokens, absolute
    int whole;                  // the run holds all of the item
    long long item0, item1, next;       // numbers: the item's, and the one behind the segment
};

// Tiles that an item of a sequence counts: the most that any of its row groups can see.
__device__ __forceinline__ int att_tiles(int length, int count, int group_rows, int g, int window) {
    const int all = (length + 63) >> 6;
    if (window == 0) return all;
    const int tokens = min(count, (group_rows + g - 1) / g + 1);
    return min(all, (min(window, length) + tokens + 62) / 64 + 1);
}

template <int D, int N8, bool SPLIT, bool E4M3>
__global__ void __launch_bounds__(kAttThreads, 1) kv_attend_kernel(const __grid_constant__ KvAttend P) {
    using A = AttendPlan<D>;
    constexpr int CW = A::kCw, LB = CW / 4, NH = LB / 8, ROWS = 8 * N8, PITCH = D + 4;
    extern __shared__ __align__(128) uint8_t att_sm[];
    __shared__ __align__(8) uint64_t full[kAttWorkers][kAttMaxSlots], empty[kAttWorkers][kAttMaxSlots];
    __shared__ long long part_item[kAttWorkers * 2][2];          // first and last number of the item that a worker's first or last part belongs to; -1: none
    __shared__ int4 part_rows[kAttWorkers * 2];                 // row0, head, item_row, rows
    __shared__ const float *part_at[kAttWorkers * 2];           // where it is
    __shared__ int part_place[kAttWorkers * 2];                 // places that have a part, in order; runs of them belong to one item
    __shared__ int run_first[kAttWorkers * 2], run_last[kAttWorkers * 2], n_runs, n_parts, n_shared, last_one[2], of_step[3];
    __shared__ int2 job[kAttWorkers * 2];                       // to put together: first and number in job_from
    __shared__ int4 job_rows[kAttWorkers * 2];
    __shared__ float *job_to[kAttWorkers * 2];                  // null: the answer
    __shared__ const float *job_from[2 * kAttMaxCtas];
    __shared__ int4 step[kAttEntries];                          // the first entries of the step
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), worker = warp & 7;
    uint8_t *ring = att_sm + worker * P.slots * A::kSlot;
    uint8_t *qs = att_sm + P.workers * P.slots * A::kSlot + worker * A::q_bytes(N8, SPLIT);
    long long *prefix = reinterpret_cast<long long *>(att_sm + P.workers * (P.slots * A::kSlot + A::q_bytes(N8, SPLIT)));
    const int g_heads = P.s.heads / P.s.kv_heads;
    const int *entries = P.book + kKvHead;
    if (tid < kAttWorkers * kAttMaxSlots) {
        mbar_init(&full[tid / kAttMaxSlots][tid % kAttMaxSlots], 1);
        mbar_init(&empty[tid / kAttMaxSlots][tid % kAttMaxSlots], 1);
        mbar_fence_init();
    }
    if (tid < kAttWorkers * 2) part_item[tid][0] = -1;
    // Numbers of one head in front of each sequence. An item counts a few tiles more than it has, for what it costs to begin and end one; nothing where
    // each worker has a part of one item anyway.
    const int all_workers = static_cast<int>(gridDim.x) * P.workers, me = static_cast<int>(blockIdx.x) * P.workers + worker;
    if (warp == 0) {
        int4 e0 = lane < P.max_seqs ? *reinterpret_cast<const int4 *>(entries + lane * kKvStepWords) : make_int4(0, 0, 0, 0);      // asked for beside their number
        const int n = P.book[0];
        if (lane < kAttEntries) step[lane] = e0;
        auto entry = [&](int i) { return i < 32 ? e0 : *reinterpret_cast<const int4 *>(entries + i * kKvStepWords); };
        if (n == 1) e0 = make_int4(__shfl_sync(0xffffffffu, e0.x, 0), __shfl_sync(0xffffffffu, e0.y, 0), __shfl_sync(0xffffffffu, e0.z, 0), __shfl_sync(0xffffffffu, e0.w, 0));
        auto items_of = [&](const int4 &e) { return (static_cast<long long>(e.z) * g_heads + ROWS - 1) / ROWS; };
        long long tiles = 0;
        int most = 0;
        for (int i = n == 1 ? 0 : lane; i < n; i += 32) {
            const int4 e = entry(i);
            const int per = att_tiles(e.w, e.z, ROWS, g_heads, P.window);
            tiles += items_of(e) * per;
            most = max(most, per);
        }
        if (n > 1) {
            most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
            for (int o = 16; o; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        }
        const int more = tiles * P.s.kv_heads >= 2ll * all_workers ? 2 : 0;
        long long sum = 0;
        if (n == 1) {               // (the usual step of a single user)
            if (lane == 0) prefix[0] = 0;
            sum = tiles + items_of(e0) * more;
        }
        for (int i0 = n == 1 ? 1 : 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            long long v = 0;
            if (i < n) {
                const int4 e = entry(i);
                if (i >= 32 && i < kAttEntries) step[i] = e;
                v = items_of(e) * (att_tiles(e.w, e.z, ROWS, g_heads, P.window) + more);
            }
            long long inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            if (i < n) prefix[i] = sum + inc - v;
            sum += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) {
            prefix[n] = sum;
            of_step[0] = n;
            of_step[1] = more;
            of_step[2] = most <= 3 ? most : 1;
        }
    }
    __syncthreads();
    const int n_seq = of_step[0], extra = of_step[1];
    const long long total = prefix[n_seq] * P.s.kv_heads;
    if (total == 0) return;
    // To put parts together costs as much as two or three tiles do: items of up to three stay whole where there are not enough of them for all workers.
    // (300 tokens, five tiles: 16.8 us whole, 12.7 shared; 131, three: 9.0 whole, 10.5 shared.)
    const long long even = (total + all_workers - 1) / all_workers, chunk = max(even, static_cast<long long>(of_step[2])), cta_chunk = chunk * P.workers;
    if (blockIdx.x * cta_chunk >= total) return;
    const long long begin = worker < P.workers ? min(me * chunk, total) : total, end = min(begin + chunk, total);
    const bool small = total < (1ll << 31);             // numbers that 32 bits hold are divided in 32 bits

    auto segment = [&](long long at) {
        AttSegment s;
        int lo = 0, hi = n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] * P.s.kv_heads <= at) lo = mid;
            else hi = mid - 1;
        }
        const int4 e = lo < kAttEntries ? step[lo] : *reinterpret_cast<const int4 *>(entries + lo * kKvStepWords);
        s.seq = e.x, s.row0 = e.y, s.count = e.z, s.length = e.w;
        const int per_item = att_tiles(s.length, s.count, ROWS, g_heads, P.window) + extra;
        const long long per_head = prefix[lo + 1] - prefix[lo], base = prefix[lo] * P.s.kv_heads, in = at - base;
        auto over = [&](long long a, long long b) { return small ? static_cast<int>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : static_cast<int>(a / b); };
        s.head = over(in, per_head);
        const int group = over(in - s.head * per_head, per_item);
        s.item0 = base + s.head * per_head + static_cast<long long>(group) * per_item;
        s.item1 = s.item0 + per_item;
        s.item_row = group * ROWS;
        s.rows = min(ROWS, s.count * g_heads - s.item_row);
        s.next = min(s.item1, end);
        s.whole = s.item0 >= begin && s.item1 <= end;
        const int pos0 = s.length - s.count + s.item_row / g_heads, pos1 = s.length - s.count + (s.item_row + s.rows - 1) / g_heads;
        const int low = P.window ? max(0, pos0 - P.window + 1) >> 6 : 0, high = (pos1 >> 6) + 1;
        s.lo = min(low + max(0, static_cast<int>(at - s.item0) - extra), high);
        s.hi = min(low + max(0, static_cast<int>(s.next - s.item0) - extra), high);
        return s;
    };

    if (warp >= kAttWorkers) {
        // ---- copies: lane 4 j + i looks up sub-block i of the j-th of eight tiles
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAttRegsLess));
        int slot = 0;
        uint32_t par = 1;
        const int shift = P.s.page_shift, grain = min(shift, 6), subs = 1 << (grain - 4);      // a copy is a page's tokens, 64 at most
        const uint32_t bytes = static_cast<uint32_t>(D) << grain;
        uint64_t *fu = full[worker], *em = empty[worker];
#pragma unroll 1
        for (long long at = begin; at < end;) {
            const AttSegment s = segment(at);
            at = s.next;
            const int *table = P.table + static_cast<size_t>(s.seq) * P.s.max_pages;
            const int last_sub = (s.length - 1) >> 4;
            const uint8_t *src = nullptr;
            float2 sc = make_float2(0.0f, 0.0f);
            auto look_up = [&](int tile0) {
                const int sub = min(4 * tile0 + lane, last_sub);            // behind the last one: the last one again, whose tokens are not seen twice
                const int page = table[sub >> (shift - 4)];
                src = P.pool + static_cast<size_t>(page) * kv_page_bytes(P.s) + s.head * kv_head_bytes(P.s) +
                      (sub & ((1 << (shift - 4)) - 1) & ~(subs - 1)) * kv_sub_bytes(D);
                sc = *reinterpret_cast<const float2 *>(P.scales + (static_cast<size_t>(page) * P.s.kv_heads + s.head) * 2);
            };
            if (s.lo < s.hi) look_up(s.lo);
#pragma unroll 1
            for (int t0 = s.lo; t0 < s.hi; t0 += 8) {
                const uint8_t *now = src;
                // (of a scale of 0, nothing but zeros, the logarithm of the least one: it costs no other weight its place)
                const float4 mine = make_float4(sc.x, log2f(fmaxf(sc.y, kKvLeastScale)), static_cast<float>(1 << kAttScale) * sc.y, 0.0f);
                if (t0 + 8 < s.hi) look_up(t0 + 8);
#pragma unroll 1
                for (int j = 0; j < 8 && t0 + j < s.hi; ++j) {
                    const bool copies = (lane >> 2) == j && (lane & (subs - 1)) == 0;
                    const int i = lane & 3;
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv) {
                        att_wait(&em[slot], par, P.status);
                        uint8_t *dst = ring + slot * A::kSlot;
                        if (kv == 0 && (lane >> 2) == j) *reinterpret_cast<float4 *>(dst + 64 * D + i * 16) = mine;
                        __syncwarp();
                        if (lane == 4 * j) mbar_expect_tx(&fu[slot], 64 * D);
                        __syncwarp();
                        if (copies) bulk_load(dst + i * 16 * D, now + kv * kv_half_bytes(P.s), bytes, &fu[slot]);
                        if (++slot == P.slots) {
                            slot = 0;
                            par ^= 1;
                        }
                    }
                }
            }
        }
        // No copy outlives the block, not where a worker's wait ran out either: the last fill of each slot (of this turn of the ring, or of the one before;
        // of none where the ring was never full, and that wait is over at once).
#pragma unroll 1
        for (int i = 0; i < P.slots; ++i) att_wait(&fu[i], i < slot ? par ^ 1 : par, P.status);
        return;
    }

    // ---- the warps that compute
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAttRegsMore));
    const int g = lane >> 2, t = lane & 3;
    int slot = 0;
    uint32_t par = 0;
    uint64_t *fu = full[worker], *em = empty[worker];
    auto pass_on = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&em[slot]);
        if (++slot == P.slots) {
            slot = 0;
            par ^= 1;
        }
    };
#pragma unroll 1
    for (long long at = begin; at < end;) {
        const AttSegment s = segment(at);
        const bool first_part = at == begin;
        at = s.next;
        // q -> fragments: [8 rows][D / CW][half of LB][lane][8 elements], hi, then lo. A lane brings a quarter of row lane / 4.
        float mul[N8][2];
        __syncwarp();
#pragma unroll
        for (int n = 0; n < N8; ++n) {
            const int r = 8 * n + g, row = s.item_row + r;
            const size_t src = static_cast<size_t>(s.row0 + row / g_heads) * P.q_stride + (static_cast<size_t>(s.head) * g_heads + row % g_heads) * D + t * (D / 4);
            float x[D / 4];
            // (the type is asked for once: asked for at each element, every load would be waited for by itself)
            auto load = [&](const auto *q) {
                using R = std::remove_const_t<std::remove_pointer_t<decltype(q)>>;
                constexpr int N = 16 / sizeof(R);
                if (P.vec) {
                    uint4 u[D / 4 / N];
#pragma unroll
                    for (int i = 0; i < D / 4 / N; ++i) u[i] = reinterpret_cast<const uint4 *>(q + src)[i];
#pragma unroll
                    for (int i = 0; i < D / 4; ++i) x[i] = static_cast<float>(reinterpret_cast<const R *>(&u[i / N])[i % N]);
                } else {
#pragma unroll
                    for (int i = 0; i < D / 4; ++i) x[i] = static_cast<float>(q[src + i]);
                }
            };
#pragma unroll
            for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
            if (r < s.rows) {
                if (P.type == kRowsF32) load(static_cast<const float *>(P.q));
                else if (P.type == kRowsF16) load(static_cast<const __half *>(P.q));
                else load(static_cast<const __nv_bfloat16 *>(P.q));
            }
            __syncwarp();
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = top > 0.0f ? max(-100, min(128, static_cast<int>(__float_as_uint(top) >> 23) - 126)) - 15 : 0, e1 = e / 2, e2 = e - e1;
            const float up = __uint_as_float((127 + e1) << 23), up2 = __uint_as_float((127 + e2) << 23), down = __uint_as_float((127 - e1) << 23),
                        down2 = __uint_as_float((127 - e2) << 23), mine = P.scale_log2 * up * up2;
            mul[n][0] = __shfl_sync(0xffffffffu, mine, 8 * t);
            mul[n][1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
#pragma unroll
            for (int i = 0; i < D / 4; i += 8) {
                const int d = t * (D / 4) + i, kk = d % CW;
                uint4 *to = reinterpret_cast<uint4 *>(qs) + ((n * (D / CW) + d / CW) * NH + kk % LB / 8) * 32 + g * 4 + kk / LB;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = x[i + 2 * j] * down * down2, b = x[i + 2 * j + 1] * down * down2;
                    hi[j] = half_pair(a, b);
                    if (SPLIT) lo[j] = half_rest(a, b, hi[j]);
                }
                to[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (SPLIT) to[ROWS * D / 8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        __syncwarp();
        float o[N8][D / 16][4], m[N8][2], l[N8][2];
        int pos[N8][2];
        const int start = s.length - s.count, last_row = s.item_row + s.rows - 1, pos_lo = start + s.item_row / g_heads, pos_hi = start + last_row / g_heads;
#pragma unroll
        for (int n = 0; n < N8; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[n][i] = kAttFloor;
                l[n][i] = 0.0f;
                pos[n][i] = start + min(s.item_row + 8 * n + 2 * t + i, last_row) / g_heads;
            }
        }
#pragma unroll 1
        for (int tile = s.lo; tile < s.hi; ++tile) {
            // tokens x rows: x[n][b][c] is token 16 b + g + 8 (c >> 1) of the tile, row 8 n + 2 t + (c & 1)
            float x[N8][4][4];
#pragma unroll
            for (int n = 0; n < N8; ++n)
#pragma unroll
                for (int b = 0; b < 4; ++b) x[n][b][0] = x[n][b][1] = x[n][b][2] = x[n][b][3] = 0.0f;
            att_wait(&fu[slot], par, P.status);
            const uint8_t *kp = ring + slot * A::kSlot + g * CW + t * LB;
            const uint4 *qp = reinterpret_cast<const uint4 *>(qs) + lane;
#pragma unroll
            for (int c = 0; c < D / CW; ++c) {
                uint4 qh[N8][NH], ql[SPLIT ? N8 : 1][NH];
#pragma unroll
                for (int n = 0; n < N8; ++n)
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        qh[n][h] = qp[((n * (D / CW) + c) * NH + h) * 32];
                        if constexpr (SPLIT) ql[n][h] = qp[((n * (D / CW) + c) * NH + h) * 32 + ROWS * D / 8];
                    }
                // (the four sub-blocks in turn at each step: products in a row on the same sums would wait for one another)
                uint32_t w0[4][LB / 4], w1[4][LB / 4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const uint8_t *p = kp + b * 16 * D + c * 16 * CW;
                    if constexpr (LB == 16) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(p), v = *reinterpret_cast<const uint4 *>(p + 8 * CW);
                        w0[b][0] = u.x, w0[b][1] = u.y, w0[b][2] = u.z, w0[b][3] = u.w;
                        w1[b][0] = v.x, w1[b][1] = v.y, w1[b][2] = v.z, w1[b][3] = v.w;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2 *>(p), v = *reinterpret_cast<const uint2 *>(p + 8 * CW);
                        w0[b][0] = u.x, w0[b][1] = u.y;
                        w1[b][0] = v.x, w1[b][1] = v.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < LB / 4; ++w)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        uint32_t a0, a1, a2, a3;
                        kv_halves<E4M3>(w0[b][w], a0, a2);
                        kv_halves<E4M3>(w1[b][w], a1, a3);
#pragma unroll
                        for (int n = 0; n < N8; ++n) {
                            const uint4 q = qh[n][w >> 1];
                            mma_f16(x[n][b], a0, a1, a2, a3, w & 1 ? q.z : q.x, w & 1 ? q.w : q.y);
                            if constexpr (SPLIT) {
                                const uint4 r = ql[n][w >> 1];
                                mma_f16(x[n][b], a0, a1, a2, a3, w & 1 ? r.z : r.x, w & 1 ? r.w : r.y);
                            }
                        }
                    }
            }
            float4 sc[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) sc[b] = *reinterpret_cast<const float4 *>(ring + slot * A::kSlot + 64 * D + b * 16);
            pass_on();
            const int first = tile * 64;
            if (first + 63 > pos_lo || (P.window && first <= pos_hi - P.window)) {
#pragma unroll
                for (int n = 0; n < N8; ++n)
#pragma unroll
                    for (int b = 0; b < 4; ++b)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int token = first + 16 * b + g + 8 * (c >> 1), at_row = pos[n][c & 1];
                            if (token > at_row || (P.window && token <= at_row - P.window)) x[n][b][c] = -INFINITY;
                        }
            }
            uint32_t ph[N8][4][2], pl[SPLIT ? N8 : 1][4][2];
            float f[N8][2];
#pragma unroll
            for (int n = 0; n < N8; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = kAttFloor;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        // (a scale of 0 makes every product 0; what is masked must not become 0 times -inf)
                        const float c = fmaxf(mul[n][i] * sc[b].x, 1e-37f);
                        top = fmaxf(top, fmaf(fmaxf(x[n][b][i], x[n][b][2 + i]), c, sc[b].y));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float now = fmaxf(m[n][i], top);
                    const float half_way = ex2(0.5f * (m[n][i] - now)), off = static_cast<float>(kAttTop - kAttScale) - now;
                    f[n][i] = half_way * half_way;
                    m[n][i] = now;
                    float sum = l[n][i] * half_way * half_way;         // (what is nothing beside the sums now may be something in the denominator)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const float c = fmaxf(mul[n][i] * sc[b].x, 1e-37f), e0 = ex2(fmaf(x[n][b][i], c, off)), e1 = ex2(fmaf(x[n][b][2 + i], c, off));
                        sum += e0 + e1;
                        x[n][b][i] = e0 * sc[b].z;
                        x[n][b][2 + i] = e1 * sc[b].z;
                    }
                    l[n][i] = sum;
                }
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t hi = half_pair(x[n][b][2 * h], x[n][b][2 * h + 1]);
                        ph[n][b][h] = transposed(hi);
                        if constexpr (SPLIT) pl[n][b][h] = transposed(half_rest(x[n][b][2 * h], x[n][b][2 * h + 1], hi));
                    }
            }
            att_wait(&fu[slot], par, P.status);
            const uint4 *vp = reinterpret_cast<const uint4 *>(ring + slot * A::kSlot) + lane;
            // A tile's sums are made apart and added in F32: a tensor core cuts its sums off, low by 6e-9 of themselves for each token that they hold.
            constexpr int KB = D / 32 < 2 ? 1 : D / 32 % 2 ? 3 : 2;          // 32 elements each; at once, for products that do not wait for one another
#pragma unroll
            for (int k0 = 0; k0 < D / 32; k0 += KB) {
                float y[KB][N8][2][4];
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int k = 0; k < KB; ++k) {
                        const uint4 v = vp[b * D + (k0 + k) * 32];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t a0, a1, a2, a3;
                            kv_halves<E4M3>(j ? v.z : v.x, a0, a2);
                            kv_halves<E4M3>(j ? v.w : v.y, a1, a3);
#pragma unroll
                            for (int n = 0; n < N8; ++n) {
                                if (b == 0) mma_f16_first(y[k][n][j], a0, a1, a2, a3, ph[n][b][0], ph[n][b][1]);
                                else mma_f16(y[k][n][j], a0, a1, a2, a3, ph[n][b][0], ph[n][b][1]);
                                if constexpr (SPLIT) mma_f16(y[k][n][j], a0, a1, a2, a3, pl[n][b][0], pl[n][b][1]);
                            }
                        }
                    }
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int n = 0; n < N8; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[n][2 * (k0 + k) + j][c] = fmaf(o[n][2 * (k0 + k) + j][c], f[n][c & 1], y[k][n][j][c]);
            }
            pass_on();
        }
        // ---- the item's end, or this worker's part of it
        const int place = worker * 2 + (first_part ? 0 : 1);
        // the worker's last part: its ring is free, and holds it
        const bool here = at >= end;
        float *part = here ? reinterpret_cast<float *>(ring) : P.part + static_cast<size_t>(me) * kAttMaxRows * PITCH;
#pragma unroll
        for (int n = 0; n < N8; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float den = l[n][i];
                den += __shfl_xor_sync(0xffffffffu, den, 4);
                den += __shfl_xor_sync(0xffffffffu, den, 8);
                den += __shfl_xor_sync(0xffffffffu, den, 16);
                const int r = 8 * n + 2 * t + i, row = s.item_row + r;
                if (r >= s.rows) continue;
                if (s.whole) {
                    const float inv = kAttUnit / den;
                    const size_t to = static_cast<size_t>(s.row0 + row / g_heads) * P.out_stride + (static_cast<size_t>(s.head) * g_heads + row % g_heads) * D + g;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        row_store(P.out, P.type, to + 16 * k, o[n][k][i] * inv);
                        row_store(P.out, P.type, to + 16 * k + 8, o[n][k][2 + i] * inv);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        part[r * PITCH + 16 * k + g] = o[n][k][i];
                        part[r * PITCH + 16 * k + 8 + g] = o[n][k][2 + i];
                    }
                    if (g == 0) *reinterpret_cast<float2 *>(part + r * PITCH + D) = make_float2(m[n][i], den);
                }
            }
        if (!s.whole && lane == 0) {
            part_item[place][0] = s.item0;
            part_item[place][1] = s.item1;
            part_rows[place] = make_int4(s.row0, s.head, s.item_row, s.rows);
            part_at[place] = part;
        }
    }

    // ---- parts of the CTA's workers: runs of places that belong to one item
    __threadfence_block();
    att_bar();
    if (warp == 0) {
        const long long item = lane < kAttWorkers * 2 ? part_item[lane][0] : -1;
        const unsigned there = __ballot_sync(0xffffffffu, item >= 0), in_front = there & ((1u << lane) - 1u);
        const long long before = __shfl_sync(0xffffffffu, item, in_front ? 31 - __clz(in_front) : lane);
        const unsigned starts = __ballot_sync(0xffffffffu, item >= 0 && (in_front == 0u || before != item));
        const unsigned behind = there & ~((2u << lane) - 1u);
        const int run = __popc(starts & ((2u << lane) - 1u)) - 1, rank = __popc(in_front);
        if (item >= 0) part_place[rank] = lane;
        if (starts >> lane & 1u) run_first[run] = rank;
        if (item >= 0 && (behind == 0u || (starts >> (__ffs(behind) - 1) & 1u))) run_last[run] = rank;
        if (lane == 0) {
            n_runs = __popc(starts);
            n_parts = __popc(there);
            n_shared = 0;
            last_one[0] = last_one[1] = -1;
        }
    }
    att_bar();
    const int runs = n_runs;
    if (runs == 0) return;
    const long long cta0 = blockIdx.x * cta_chunk, cta1 = min(cta0 + cta_chunk, total);
    constexpr int V = D / 4;
    auto cta_of = [&](long long at) { return small ? static_cast<int>(static_cast<uint32_t>(at) / static_cast<uint32_t>(cta_chunk)) : static_cast<int>(at / cta_chunk); };
    // the CTA's parts of its runs: answers, or a part of the first or the last run, which others may hold parts of too
    if (tid < runs) {
        const int p0 = part_place[run_first[tid]];
        const long long item0 = part_item[p0][0], item1 = part_item[p0][1];
        const bool ours = item0 >= cta0 && item1 <= cta1;
        job[tid] = make_int2(run_first[tid], run_last[tid] - run_first[tid] + 1);
        job_rows[tid] = part_rows[p0];
        job_to[tid] = ours ? nullptr : P.cta_part + (static_cast<size_t>(blockIdx.x) * 2 + (item0 <= cta0 ? 0 : 1)) * kAttMaxRows * PITCH;
        if (!ours) atomicAdd_block(&n_shared, 1);
    }
    if (tid < n_parts) job_from[tid] = part_at[part_place[tid]];
    att_bar();
    // Parts are put together twice: the workers' of a CTA, then the CTAs' of an item, by the last of them to arrive. One loop serves both: code that an SM
    // has not run yet costs far more than what it does (two copies: 13 us for the second one).
    int jobs = runs;
#pragma unroll 1
    for (int turn = 0;; ++turn) {
#pragma unroll 1
        for (int i = tid; i < jobs * ROWS * V; i += kAttWorkers * 32) {
            const int j = i / (ROWS * V), r = i / V % ROWS, c = i % V * 4, n = job[j].y;
            const int4 rw = job_rows[j];
            if (r >= rw.w) continue;
            const float *const *from = job_from + job[j].x;
            float top = kAttFloor, den = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (int k0 = 0; k0 < n; k0 += 4) {
                float4 y[4];
                float2 z[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {           // (volatile: what other warps, or CTAs, have written)
                    const float *p = from[min(k0 + k, n - 1)] + r * PITCH;
                    asm volatile("ld.volatile.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[k].x), "=f"(y[k].y), "=f"(y[k].z), "=f"(y[k].w) : "l"(p + c));
                    asm volatile("ld.volatile.v2.f32 {%0, %1}, [%2];" : "=f"(z[k].x), "=f"(z[k].y) : "l"(p + D));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k0 + k >= n) break;
                    const float both = fmaxf(top, z[k].x), ha = ex2(0.5f * (top - both)), hb = ex2(0.5f * (z[k].x - both)), fa = ha * ha, fb = hb * hb;
                    top = both;
                    den = den * ha * ha + z[k].y * hb * hb;
                    sum.x = sum.x * fa + y[k].x * fb, sum.y = sum.y * fa + y[k].y * fb, sum.z = sum.z * fa + y[k].z * fb, sum.w = sum.w * fa + y[k].w * fb;
                }
            }
            if (float *to = job_to[j]) {
                __stcg(reinterpret_cast<float4 *>(to + r * PITCH + c), sum);
                if (c == 0) __stcg(reinterpret_cast<float2 *>(to + r * PITCH + D), make_float2(top, den));
            } else {
                const int row = rw.z + r;
                const size_t to0 = static_cast<size_t>(rw.x + row / g_heads) * P.out_stride + (static_cast<size_t>(rw.y) * g_heads + row % g_heads) * D + c;
                const float inv = kAttUnit / den;
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    row_store(P.out, P.type, to0 + k, sum.x * inv);
                    sum.x = sum.y, sum.y = sum.z, sum.z = sum.w;
                }
            }
        }
        if (turn > 0 || n_shared == 0) return;
        __threadfence();
        att_bar();
        if (tid < 2) {
            const int run = tid == 0 ? 0 : runs - 1;
            if (job_to[run] && (tid == 0 || runs > 1)) {
                const int p0 = part_place[run_first[run]];
                const int c0 = cta_of(part_item[p0][0]), c1 = cta_of(part_item[p0][1] - 1);
                const unsigned before = atomicAdd(P.arrived + c0, 1u);
                if (before == static_cast<unsigned>(c1 - c0)) {
                    P.arrived[c0] = 0u;
                    last_one[tid] = run;
                }
                __threadfence();
            }
        }
        att_bar();
        // the jobs of the second turn: one for each run that this CTA was the last to bring its part of
        jobs = 0;
        int at = 0;
        for (int w = 0; w < 2; ++w) {
            const int run = last_one[w];
            if (run < 0) continue;
            const int p0 = part_place[run_first[run]];
            const long long item0 = part_item[p0][0];
            const int c0 = cta_of(item0), n = cta_of(part_item[p0][1] - 1) - c0 + 1;
            for (int k = tid; k < n; k += kAttWorkers * 32)
                job_from[at + k] = P.cta_part + (static_cast<size_t>(c0 + k) * 2 + (item0 <= (c0 + k) * cta_chunk ? 0 : 1)) * kAttMaxRows * PITCH;
            if (tid == 0) {
                job[jobs] = make_int2(at, n);
                job_rows[jobs] = part_rows[p0];
                job_to[jobs] = nullptr;
            }
            ++jobs;
            at += n;
        }
        if (jobs == 0) return;
        att_bar();
    }
}

}  // namespace wd
