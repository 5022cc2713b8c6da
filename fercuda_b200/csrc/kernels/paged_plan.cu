// The plan of a serving step over a paged key-value cache: which sequences get
// the rows they ask for, which pages they take and give back, and which
// sequence, position and slot each row of the step's activation has.
//
// With P slots a page, sequence b asks for ask_b = max(0, ceil((lengths + counts)
// / P) - held) pages. Sums over the sequences before decide: b is granted where
// ask_b is 0 or the sum up to and with b is at most what the ring of free pages
// has, so granted sequences take pages from the ring's beginning at the sum of
// what was asked before them. Pages go back behind the ring's end, which no
// taken page overlaps as long as a page is in one place.
//
// A few bytes a sequence and 12 a row: the pass is bound by the latency of
// three dependent steps (sums, pages, rows). One cluster of CTAs does them all,
// so that two cluster barriers stand where launches would: each thread has a few
// neighbouring sequences, the sums are a scan over the cluster's threads, page
// ids are moved by whole warps, and a row finds its sequence by a search among
// every few sequences' first rows in shared memory (a thread's next rows walk on from
// there, over sequences without rows one by one). One CTA does it where there
// are few rows and sequences; where there are many rows a second launch spreads
// them over the GPU (1024 requests with 236000 rows: 30 us by the cluster, 21 so).
#include "paged.cuh"
#include "pdl.cuh"

#include <cooperative_groups.h>

#include <climits>
#include <cstdint>

namespace cg = cooperative_groups;

namespace {

constexpr int kCtas = 8;             // of a cluster
constexpr int kStarts = 4096;        // first rows in shared memory
constexpr int kFewSequences = 256, kFewRows = 1024;     // what a small CTA does alone
constexpr int kOneRows = 4096;       // rows that a CTA fills alone
constexpr int kManyRows = 16384;     // rows with a launch of their own
constexpr int kRowThreads = 256;

struct PlanParams {
    int32_t* table;
    const int32_t *lengths, *counts, *held, *seen;
    int32_t* ring;
    const int32_t* state;
    int32_t *new_held, *new_state, *offsets, *sequences, *positions, *slots;
    int batch, max_pages, pages, shift, rows;
    int each, across;   // sequences a thread, and lanes of a warp that have some
    uint32_t* err;
};

// Sums of what the sequences before a place ask for, get as rows and give back.
struct Sums {
    long long ask, rows, give;
    __device__ __forceinline__ void add(const Sums& o) { ask += o.ask, rows += o.rows, give += o.give; }
};

// One sequence's part, from its numbers alone.
struct Request {
    int length, count, held, keep, need;
    bool bad;
    __device__ __forceinline__ Request(const PlanParams& p, int b) {
        const int most = p.max_pages << p.shift, up = (1 << p.shift) - 1;
        length = p.lengths[b], count = p.counts[b], held = p.held[b];
        bad = length < 0 || length > most || count < 0 || held < 0 || held > p.max_pages;
        length = min(max(length, 0), most);
        count = max(count, 0);
        held = min(max(held, 0), p.max_pages);
        if (count > most - length) bad = true, count = 0;   // more than its row of the table holds: refused
        keep = (length + up) >> p.shift;
        need = (length + count + up) >> p.shift;
    }
    __device__ __forceinline__ int ask() const { return max(need - held, 0); }
};

__device__ __forceinline__ long long shfl_up(long long v, int off) { return __shfl_up_sync(0xffffffffu, v, off); }

// The sums of the threads before this one over the whole cluster, and the total.
template <int CTAS, int THREADS>
__device__ __forceinline__ Sums scan(Sums mine, Sums (&s_warp)[32], Sums& s_cta, Sums& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    Sums x = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const Sums y{shfl_up(x.ask, off), shfl_up(x.rows, off), shfl_up(x.give, off)};
        if (lane >= off) x.add(y);
    }
    if (lane == 31) s_warp[w] = x;
    __syncthreads();
    Sums before{}, all{};
    {
        Sums y = lane < THREADS / 32 ? s_warp[lane] : Sums{};
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const Sums z{shfl_up(y.ask, off), shfl_up(y.rows, off), shfl_up(y.give, off)};
            if (lane >= off) y.add(z);
        }
        all = Sums{__shfl_sync(0xffffffffu, y.ask, 31), __shfl_sync(0xffffffffu, y.rows, 31), __shfl_sync(0xffffffffu, y.give, 31)};
        const Sums e{__shfl_sync(0xffffffffu, y.ask, max(w - 1, 0)), __shfl_sync(0xffffffffu, y.rows, max(w - 1, 0)),
                     __shfl_sync(0xffffffffu, y.give, max(w - 1, 0))};
        if (w > 0) before = e;
    }
    before.add(Sums{x.ask - mine.ask, x.rows - mine.rows, x.give - mine.give});
    if constexpr (CTAS > 1) {
        const cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) s_cta = all;
        cluster.sync();
        const int rank = static_cast<int>(cluster.block_rank());
        all = Sums{};
        for (int i = 0; i < CTAS; ++i) {
            const Sums v = *cluster.map_shared_rank(&s_cta, i);
            if (i < rank) before.add(v);
            all.add(v);
        }
        // the next scan writes another s_cta, and no CTA leaves before the kernel's last barrier
    }
    __syncthreads();
    total = all;
    return before;
}

// Place i of the ring of n that begins at `first`.
__device__ __forceinline__ size_t ring_at(int first, unsigned i, int n) {
    const unsigned at = static_cast<unsigned>(first) + i;
    return at >= static_cast<unsigned>(n) ? at - n : at;
}

// Rows from r0 on, four a thread, step apart; s_start: first rows of every few sequences.
__device__ __forceinline__ void fill_rows(const PlanParams& p, int* s_start, int starts_most, long long r0, long long step_rows,
                                          long long total);

template <int CTAS, int THREADS>
__global__ void __launch_bounds__(THREADS) plan(const PlanParams p, const int fill) {
    __shared__ Sums s_warp[32], s_cta[2];
    __shared__ int s_start[CTAS > 1 ? kStarts : kFewSequences];
    const int t = threadIdx.x, lane = t & 31;
    int rank = 0;
    if constexpr (CTAS > 1) rank = static_cast<int>(cg::this_cluster().block_rank());
    const int thread = rank * THREADS + t;
    fer::dev::pdl_begin();

    // a ring that cannot be gives and takes nothing
    int first = p.state[0], free = p.state[1];
    const bool broken = first < 0 || first >= p.pages || free < 0 || free > p.pages;
    bool bad = broken;
    const int room = broken ? 0 : p.pages - free;
    const int kept_first = first, kept_free = free;
    if (broken) first = free = 0;
    // few sequences are spread over all warps, as a warp moves the page ids of one at a time
    const long long place = (static_cast<long long>(thread >> 5) * p.across + lane) * p.each;
    const int b0 = lane < p.across ? static_cast<int>(min(place, static_cast<long long>(p.batch))) : p.batch;
    const int b1 = min(p.batch, b0 + p.each);

    Sums mine{}, total{};
    for (int b = b0; b < b1; ++b) mine.ask += Request(p, b).ask();
    const Sums asked = scan<CTAS, THREADS>(mine, s_warp, s_cta[0], total);
    const auto granted = [&](long long before, int ask) { return ask == 0 || before + ask <= free; };
    // what a sequence holds afterwards; where the ring cannot be, nothing goes back
    const auto pages_after = [&](const Request& r, bool on) { return broken ? r.held : on ? r.need : min(r.held, r.keep); };
    mine = Sums{};
    {
        long long before = asked.ask;
        for (int b = b0; b < b1; ++b) {
            const Request r(p, b);
            const bool on = granted(before, r.ask());
            before += r.ask();
            bad = bad || r.bad;
            mine.ask += on ? r.ask() : 0;
            mine.rows += on ? r.count : 0;
            mine.give += r.held - min(r.held, pages_after(r, on));
        }
    }
    Sums at = scan<CTAS, THREADS>(mine, s_warp, s_cta[1], total);
    if (thread == 0) {
        if (broken) {
            p.new_state[0] = kept_first, p.new_state[1] = kept_free;
        } else {
            const long long given = min(total.give, static_cast<long long>(room));
            if (given < total.give) bad = true;
            p.new_state[0] = static_cast<int>(ring_at(first, static_cast<unsigned>(total.ask), p.pages));
            p.new_state[1] = static_cast<int>(free - total.ask + given);
        }
        p.offsets[0] = 0;
        if (total.rows > p.rows) bad = true;
    }

    // offsets and pages; a warp moves one sequence's page ids at a time
    long long before = asked.ask;
    for (int i = 0; i < p.each; ++i) {
        const int b = b0 + i;   // of lanes without one behind the last
        int held = 0, now = 0;
        long long take_at = 0, give_at = 0;
        if (b < b1) {
            const Request r(p, b);
            const bool on = granted(before, r.ask());
            take_at = before, give_at = at.give;
            before += r.ask();
            held = r.held;
            now = pages_after(r, on);
            at.rows += on ? r.count : 0;
            at.give += max(held - now, 0);
            if (at.rows > INT_MAX) bad = true;
            p.offsets[b + 1] = static_cast<int>(min(at.rows, static_cast<long long>(INT_MAX)));
            p.new_held[b] = now;
        }
        unsigned busy = __ballot_sync(0xffffffffu, held != now);
        while (busy) {
            const int src = __ffs(busy) - 1;
            busy &= busy - 1;
            const int h = __shfl_sync(0xffffffffu, held, src), n = __shfl_sync(0xffffffffu, now, src);
            const long long ta = __shfl_sync(0xffffffffu, take_at, src), ga = __shfl_sync(0xffffffffu, give_at, src);
            int32_t* const row = p.table + static_cast<size_t>(__shfl_sync(0xffffffffu, b, src)) * p.max_pages;
            for (int j = h + lane; j < n; j += 32) {
                const int id = p.ring[ring_at(first, static_cast<unsigned>(ta + (j - h)), p.pages)];
                bad = bad || static_cast<unsigned>(id) >= static_cast<unsigned>(p.pages);
                row[j] = id;
            }
            for (int j = n + lane; j < h; j += 32) {
                const long long to = ga + (j - n);
                if (to >= room) break;   // no room: reported above
                const int id = row[j];
                bad = bad || static_cast<unsigned>(id) >= static_cast<unsigned>(p.pages);
                p.ring[ring_at(first, static_cast<unsigned>(free + to), p.pages)] = id;
            }
        }
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    // offsets and page ids are there for every CTA; and each has read the others' shared memory
    if constexpr (CTAS > 1) cg::this_cluster().sync();
    else __syncthreads();
    if (fill) fill_rows(p, s_start, CTAS > 1 ? kStarts : kFewSequences, 4ll * thread, 4ll * CTAS * THREADS, total.rows);
}

__device__ __forceinline__ void fill_rows(const PlanParams& p, int* s_start, int starts_most, long long r0, long long step_rows,
                                          long long total) {
    const int t = threadIdx.x, step = (p.batch + starts_most - 1) / starts_most, starts = (p.batch + step - 1) / step;
    for (int i = t; i < starts; i += blockDim.x) s_start[i] = __ldcg(p.offsets + static_cast<size_t>(i) * step);
    __syncthreads();
    const bool wide = (reinterpret_cast<uintptr_t>(p.sequences) | reinterpret_cast<uintptr_t>(p.positions) |
                       reinterpret_cast<uintptr_t>(p.slots)) % 16 == 0;
    const int rows = static_cast<int>(min(total, static_cast<long long>(p.rows)));
    for (; r0 < p.rows; r0 += step_rows) {
        int seq[4], pos[4], slot[4];
        int b = -1, begin = 0, end = 0, length = 0, seen = 0, base = -1, page = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            seq[e] = -1, pos[e] = 0, slot[e] = -1;
            const long long r = r0 + e;
            if (r >= rows) continue;
            if (r >= end) {
                if (b < 0) {
                    int lo = 0, hi = starts;   // the last of every `step` sequences that starts at or before r
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (s_start[mid] <= r) lo = mid;
                        else hi = mid;
                    }
                    b = lo * step;
                    begin = s_start[lo];
                } else {
                    ++b;
                    begin = end;
                }
                for (end = __ldcg(p.offsets + b + 1); r >= end; end = __ldcg(p.offsets + b + 1)) ++b, begin = end;
                length = min(max(p.lengths[b], 0), p.max_pages << p.shift);
                seen = p.positions && p.seen ? p.seen[b] : length;
                base = -1;
            }
            const int i = static_cast<int>(r) - begin, s = length + i;
            seq[e] = b;
            pos[e] = seen + i;
            if (p.slots) {
                if (s >> p.shift != base) {
                    base = s >> p.shift;
                    page = __ldcg(p.table + static_cast<size_t>(b) * p.max_pages + base);
                }
                if (static_cast<unsigned>(page) < static_cast<unsigned>(p.pages))
                    slot[e] = (page << p.shift) + (s & ((1 << p.shift) - 1));
                else fer::dev::report(p.err, fer::dev::kErrBadShape);
            }
        }
        if (wide && r0 + 4 <= p.rows) {
            if (p.sequences) *reinterpret_cast<int4*>(p.sequences + r0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
            if (p.positions) *reinterpret_cast<int4*>(p.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            if (p.slots) *reinterpret_cast<int4*>(p.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (r0 + e >= p.rows) break;
                if (p.sequences) p.sequences[r0 + e] = seq[e];
                if (p.positions) p.positions[r0 + e] = pos[e];
                if (p.slots) p.slots[r0 + e] = slot[e];
            }
        }
    }
}

// The rows of a plan whose offsets and pages are there.
__global__ void __launch_bounds__(kRowThreads) plan_rows(const PlanParams p) {
    __shared__ int s_start[kStarts];
    fer::dev::pdl_begin();
    const long long thread = static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x;
    fill_rows(p, s_start, kStarts, 4 * thread, 4ll * gridDim.x * kRowThreads, __ldcg(p.offsets + p.batch));
}

}  // namespace

extern "C" cudaError_t fer_paged_plan(const fer_paged_plan_args_t* a, uint32_t* err, cudaStream_t s) {
    if (!a || !a->page_table || !a->lengths || !a->counts || !a->held || !a->free_pages || !a->free_state || !a->new_held ||
        !a->new_free_state || !a->offsets)
        return cudaErrorInvalidValue;
    if (a->batch <= 0 || a->max_pages <= 0 || a->pages <= 0 || a->rows < 0) return cudaErrorInvalidValue;
    if (!fer::host::words_aligned({a->page_table, a->lengths, a->counts, a->held, a->seen, a->free_pages, a->free_state,
                                   a->new_held, a->new_free_state, a->offsets, a->sequences, a->positions, a->slots}))
        return cudaErrorInvalidValue;
    int shift = 3;
    while (shift < 8 && (1 << shift) != a->page_size) ++shift;
    if ((1 << shift) != a->page_size) return cudaErrorNotSupported;
    // slots of a sequence and of all pages are counted in 31 bits
    if (a->batch > 65535 || (static_cast<long long>(a->max_pages) << shift) > INT_MAX - 65536ll ||
        (static_cast<long long>(a->pages) << shift) > INT_MAX)
        return cudaErrorNotSupported;
    PlanParams p{};
    p.table = a->page_table;
    p.lengths = a->lengths;
    p.counts = a->counts;
    p.held = a->held;
    p.seen = a->seen;
    p.ring = a->free_pages;
    p.state = a->free_state;
    p.new_held = a->new_held;
    p.new_state = a->new_free_state;
    p.offsets = a->offsets;
    p.sequences = a->sequences;
    p.positions = a->positions;
    p.slots = a->slots;
    p.batch = a->batch;
    p.max_pages = a->max_pages;
    p.pages = a->pages;
    p.shift = shift;
    p.rows = a->sequences || a->positions || a->slots ? a->rows : INT_MAX;
    p.err = err;
    const int fill = a->sequences || a->positions || a->slots;
    const int alone = fill ? a->rows : 0;
    p.each = 1;
    const auto spread = [&](int warps) {
        p.across = (a->batch + warps - 1) / warps;
        if (p.across > 32) p.each = (p.across + 31) / 32, p.across = 32;
    };
    if (a->batch <= kFewSequences && alone <= kFewRows) {
        spread(kFewSequences / 32);
        return fer::host::launch_pdl(plan<1, kFewSequences>, dim3(1), dim3(kFewSequences), 0, s, p, fill);
    }
    cudaError_t e;
    if (a->batch <= kFewSequences && (alone <= kOneRows || alone > kManyRows)) {
        spread(32);
        e = fer::host::launch_pdl(plan<1, 1024>, dim3(1), dim3(1024), 0, s, p, alone > kManyRows ? 0 : fill);
    } else {
        spread(32 * kCtas);
        e = fer::host::launch_pdl_cluster(plan<kCtas, 1024>, dim3(kCtas), dim3(1024), 0, kCtas, s, p, alone > kManyRows ? 0 : fill);
    }
    if (e != cudaSuccess || alone <= kManyRows) return e;
    const int ctas = (a->rows - 1) / (4 * kRowThreads) + 1;
    return fer::host::launch_pdl(plan_rows, dim3(ctas < 4 * 148 ? ctas : 4 * 148), dim3(kRowThreads), 0, s, p);
}
