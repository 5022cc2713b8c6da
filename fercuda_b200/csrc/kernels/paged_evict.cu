// Eviction from a paged cache by accumulated attention weight.
//
// Every (sequence, key head) of n > budget slots keeps `budget` of them: a
// selection over n keys, then the move of the kept rows that lie behind the
// budget into the rows freed before it. Sources lie at or behind `budget` and
// targets before it, so all moves are independent. What has to be read is 8
// bytes a slot (weight, position), and 2 x 2 x head_dim elements a moved row.
//
// A slot's key is 32 bits: all ones for a recent one, else the weight's bits
// in an order of unsigned integers (NaN 0). Kept are the keys above a cut, and
// of the slots with exactly that key the lowest. Weights and positions are
// read once; those before the budget are copied to their new arrays as they
// pass (what is freed among them the moves overwrite, which are as many).
//
// Measured: 64 sequences x 16 heads of 64 cut from 513 to 512 slots 6.4 us
// (one chain of latencies: arrays, cut, page ids, rows); 4 sequences of up to
// 32768 x 8 heads of 128 cut to 4096 32.2 us, of which 13 us are the selection
// and 17 us the moves (16.5 us for all bytes at the copy rate).
//
// Up to 1024 slots (evict_small): a warp a head with its keys in registers,
// lane-strided, finds the cut bit by bit: at most 32 counts, no shared memory
// and no barrier, and it stops as soon as a cut leaves exactly the budget.
// What a lane frees, keeps and moves are then 32-bit masks, and only the key
// registers that hold such a slot in some lane cost a ballot. Where lengths
// are replaced in place a sequence's heads share a cluster, and its length is
// replaced once all have read it. When a head can have at most 32 moves (a
// cache that is cut back every few tokens) the warp also makes them, and one
// launch does it all.
//
// Above (evict_select): a CTA a head, or a cluster of 2 to 8 of them, with the
// keys in shared memory, and three digits of 12, 12 and 8 bits (or four of 10
// in the smaller CTAs that short heads take where there are many) counted there;
// the other CTAs' counts are read through distributed shared memory. Beyond 8
// x 32K slots the keys are made again for every pass.
//
// The moves (evict_move, or the selecting CTAs where heads come in waves): a
// warp resolves up to 32 moves at once, a lane each, then copies their rows
// with kAhead 16-byte loads a lane in flight.
#include "evict_keys.h"
#include "paged.cuh"
#include "pdl.cuh"

#include <cooperative_groups.h>

#include <atomic>
#include <cstdint>

namespace {

namespace cg = cooperative_groups;
using fer::dev::Paged;
constexpr uint32_t kAll = 0xffffffffu;
constexpr int kSmall = 1024;                 // slots that a warp's registers hold
constexpr int kSelect = 1024, kSelectFew = 256;   // threads of a selecting CTA
using fer::evict::kMostKeys;
constexpr int kCopies = 3;                   // of the first digit's counts, by lane: less contention
constexpr int kMove = 256;
constexpr int kWarpMoves = 16;
constexpr int kFusedMoves = 32;
constexpr int kFuseCtas = 2 * 148;           // selecting CTAs from which on they also move rows
constexpr int kFewDropped = 4;               // slots too many that are found one by one

struct EvictParams {
    int budget, recent, cap;     // cap: moves a (sequence, key head) can have
    int fused;                   // the selecting kernel moves rows
    int late;                    // lengths are replaced in place, by a kernel behind all of their readers
    const float* weights;
    const int32_t* positions;
    const int32_t* seen;
    int32_t* new_lengths;
    float* new_weights;
    int32_t* new_positions;
    int32_t* counts;             // [batch * kv_heads]
    int32_t* to;                 // [batch * kv_heads][cap] freed slots, ascending
    int32_t* from;               // [batch * kv_heads][cap] kept slots behind the budget, ascending
    uint32_t* err;
};

__device__ __forceinline__ uint32_t key_of(float w, int pos, long long first_recent) {
    if (pos >= first_recent) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);   // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// One (sequence, key head): its arrays.
struct Head {
    const float* w;
    const int32_t* pos;
    float* nw;
    int32_t* np;
    int32_t* to;
    int32_t* from;
};

__device__ __forceinline__ Head head_of(const Paged& c, const EvictParams& p, size_t bh) {
    const size_t at = bh * static_cast<size_t>(c.max_slots());
    return Head{p.weights + at,     p.positions + at,  p.new_weights + at,
                p.new_positions + at, p.to + bh * p.cap, p.from + bh * p.cap};
}

// Up to 32 moves of one head, move i0 + lane in each lane: their slots are
// resolved to rows, a lane each, then all lanes copy row after row.
template <int D, int kAhead>
__device__ __forceinline__ void move_rows(const Paged& c, const EvictParams& p, const Head& h, int hk, bool mine,
                                          int from, int to, int pf, int pt) {   // pf, pt: their pages, as the table has them
    constexpr int kPieces = D / 8, kRows = 32 / kPieces;   // lanes a row, rows at once
    const int lane = threadIdx.x & 31, piece = lane % kPieces;
    unsigned long long src = 0, dst = 0;
    bool good = false;
    if (mine) {
        h.nw[to] = h.w[from];
        h.np[to] = h.pos[from];
        good = c.is_page(pf) && c.is_page(pt);
        if (good) src = c.row(pf, hk, from), dst = c.row(pt, hk, to);
        else fer::dev::report(p.err, fer::dev::kErrBadShape);
    }
    const uint32_t goods = __ballot_sync(kAll, good);
    // row 2 i is the key and 2 i + 1 the value of move i
    const int rows = 2 * (32 - __clz(goods));
    for (int x0 = 0; x0 < rows; x0 += kAhead * kRows) {
        uint4 v[kAhead];
        uint16_t* at[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int x = x0 + k * kRows + lane / kPieces;
            const unsigned long long rs = __shfl_sync(kAll, src, (x >> 1) & 31), rd = __shfl_sync(kAll, dst, (x >> 1) & 31);
            at[k] = nullptr;
            if (x < rows && (goods >> (x >> 1) & 1u)) {
                uint16_t* base = static_cast<uint16_t*>(x & 1 ? c.v : c.k) + piece * 8;
                v[k] = *reinterpret_cast<const uint4*>(base + rs);
                at[k] = base + rd;
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (at[k]) *reinterpret_cast<uint4*>(at[k]) = v[k];
    }
}

__device__ __forceinline__ void copy_whole(const Head& h, int n, int t, int step) {
    for (int j = t; j < n; j += step) {
        if (h.nw != h.w) h.nw[j] = h.w[j];
        if (h.np != h.pos) h.np[j] = h.pos[j];
    }
}

// The low `n` bits, n clamped to 0 .. 32.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? kAll : n <= 0 ? 0u : (1u << n) - 1u; }

// grid (CTAs a sequence, batch), a warp a head, for max_slots <= 32 * KEYS;
// where the length is replaced in place a sequence's CTAs are a cluster. Slot
// 32 i + lane is key i of that lane.
template <int D, int KEYS>
__global__ void __launch_bounds__(256) evict_small(const Paged c, const EvictParams p) {
    __shared__ int s_to[8][kFusedMoves], s_from[8][kFusedMoves];
    const cg::cluster_group cluster = cg::this_cluster();
    const int b = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int warps = blockDim.x >> 5, step = warps * gridDim.x;
    if (blockIdx.x * warps + w < c.kv_heads) {   // the first head's arrays, and the page ids
        const Head h = head_of(c, p, static_cast<size_t>(b) * c.kv_heads + blockIdx.x * warps + w);
        if (32 * lane < c.max_slots()) {
            fer::dev::prefetch_l2(h.w + 32 * lane);
            fer::dev::prefetch_l2(h.pos + 32 * lane);
        }
        if (32 * lane < c.max_pages) fer::dev::prefetch_l2(c.table + static_cast<size_t>(b) * c.max_pages + 32 * lane);
    }
    fer::dev::pdl_begin();
    bool bad;
    const int n = c.length(b, &bad);
    if (bad && threadIdx.x == 0 && blockIdx.x == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    const long long first = static_cast<long long>(p.seen[b]) - p.recent;
    // the sequence's page ids, lane-strided, for the moves of this kernel
    constexpr int kPages = (32 * KEYS / 8 + 31) / 32;
    int pages[kPages];
    if (p.fused) {
#pragma unroll
        for (int i = 0; i < kPages; ++i) {
            pages[i] = -1;
            if (32 * i + lane < c.max_pages) pages[i] = c.table[static_cast<size_t>(b) * c.max_pages + 32 * i + lane];
        }
    }
    auto page_of = [&](int i) {
        int id = -1;
#pragma unroll
        for (int k = 0; k < kPages; ++k) {
            const int v = __shfl_sync(kAll, pages[k], i & 31);
            if (i >> 5 == k) id = v;
        }
        return id;
    };
    for (int hk = blockIdx.x * warps + w; hk < c.kv_heads; hk += step) {
        const size_t bh = static_cast<size_t>(b) * c.kv_heads + hk;
        const Head h = head_of(c, p, bh);
        if (n <= p.budget) {
            copy_whole(h, n, lane, 32);
            if (lane == 0) p.counts[bh] = 0;
            continue;
        }
        uint32_t key[KEYS];   // 0 behind the last slot
        {
            float wt[KEYS];
            int pos[KEYS];
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
                const int j = min(32 * i + lane, n - 1);
                wt[i] = h.w[j];
                pos[i] = h.pos[j];
            }
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
                const int j = 32 * i + lane;
                key[i] = j < n ? key_of(wt[i], pos[i], first) : 0u;
                if (j < p.budget) {
                    if (h.nw != h.w) h.nw[j] = wt[i];
                    if (h.np != h.pos) h.np[j] = pos[i];
                }
            }
        }
        // the largest cut with at least `budget` keys at or above it
        uint32_t cut = 0u;
        int above = n;   // keys >= cut
        if (n - p.budget <= kFewDropped) {
            // up from the least key, one value at a time
            for (uint32_t from = 0u;;) {
                uint32_t least = kAll;
#pragma unroll
                for (int i = 0; i < KEYS; ++i)
                    if (32 * i + lane < n && key[i] >= from) least = min(least, key[i]);
                least = __reduce_min_sync(kAll, least);
                int m = 0;
#pragma unroll
                for (int i = 0; i < KEYS; ++i) m += 32 * i + lane < n && key[i] == least ? 1 : 0;
                m = __reduce_add_sync(kAll, m);
                cut = least;
                if (above - m < p.budget || least == kAll) break;
                above -= m;
                from = least + 1u;
            }
        } else {
            // bit by bit, from the highest in which keys differ
            uint32_t differ = 0u, any = __shfl_sync(kAll, key[0], 0);
#pragma unroll
            for (int i = 0; i < KEYS; ++i) differ |= 32 * i + lane < n ? key[i] ^ any : 0u;
            differ = __reduce_or_sync(kAll, differ);
            const int top = 31 - __clz(differ);   // -1: all keys are alike
            cut = any & ~low_bits(top + 1);
            for (int bit = top; bit >= 0 && above != p.budget; --bit) {
                const uint32_t next = cut | 1u << bit;
                int m[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KEYS; ++i) m[i & 3] += key[i] >= next ? 1 : 0;   // next > 0: not those behind n
                const int sum = __reduce_add_sync(kAll, (m[0] + m[1]) + (m[2] + m[3]));
                if (sum >= p.budget) cut = next, above = sum;
            }
        }
        const uint32_t held = low_bits((n - lane + 31) >> 5), front = low_bits((p.budget - lane + 31) >> 5);
        uint32_t kept = 0u, equal = 0u;   // bit i: slot 32 i + lane
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            kept |= (key[i] >= cut ? 1u : 0u) << i;
            equal |= (key[i] == cut ? 1u : 0u) << i;
        }
        kept &= held;
        equal &= held;
        if (above > p.budget) {   // of the slots whose key is the cut the highest are not kept
            int drop = above - p.budget;
            for (uint32_t some = __reduce_or_sync(kAll, equal); drop > 0 && some;) {
                const int i = 31 - __clz(some);
                some &= ~(1u << i);
                const uint32_t row = __ballot_sync(kAll, equal >> i & 1u);
                if ((row >> lane & 1u) && __popc(row >> lane) <= drop) kept &= ~(1u << i);
                drop -= __popc(row);
            }
        }
        const uint32_t hole = held & front & ~kept, move = kept & ~front;
        int* to = p.fused ? s_to[w] : h.to;
        int* from = p.fused ? s_from[w] : h.from;
        int count[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t bits = e ? move : hole;
            for (uint32_t some = __reduce_or_sync(kAll, bits); some; some &= some - 1u) {
                const int i = __ffs(some) - 1;
                const uint32_t row = __ballot_sync(kAll, bits >> i & 1u);
                const int at = count[e] + __popc(row & ((1u << lane) - 1u));
                if ((bits >> i & 1u) && at < p.cap) (e ? from : to)[at] = 32 * i + lane;
                count[e] += __popc(row);
            }
        }
        const int moved = min(count[0], min(count[1], p.cap));   // all alike
        if (p.fused) {
            __syncwarp();
            const int f = lane < moved ? from[lane] : 0, g = lane < moved ? to[lane] : 0;
            move_rows<D, 8>(c, p, h, hk, lane < moved, f, g, page_of(f >> c.shift), page_of(g >> c.shift));
            __syncwarp();
        } else if (lane == 0) {
            p.counts[bh] = moved;
        }
    }
    cluster.sync();   // every head of the cluster has read the length
    if (blockIdx.x == 0 && threadIdx.x == 0) p.new_lengths[b] = min(n, p.budget);
}

// Exclusive prefix sum over the block, and the total.
template <int kWarps>
__device__ __forceinline__ int block_scan(int v, int* sh, int* total) {
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    int x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(kAll, x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[w] = x;
    __syncthreads();
    const int sum = lane < kWarps ? sh[lane] : 0;
    *total = __reduce_add_sync(kAll, sum);
    return __reduce_add_sync(kAll, lane < w ? sum : 0) + x - v;
}

// grid (cluster CTAs, kv_heads, batch). CTA r of a cluster has the slots [lo,
// hi). They are passed over in rounds of up to 32 slots a thread, shared out
// evenly; the key of slot lo + j lies at word word_of(j) of shared memory.
// Without HELD the keys of a round are made again from the arrays.
template <int D, bool HELD, int kSelect>
__global__ void __launch_bounds__(kSelect, 1024 / kSelect) evict_select(const Paged c, const EvictParams p) {
    // Digits: with two counts a word (a CTA's held keys are few enough), four
    // bins a thread, else two.
    constexpr int kWarps = kSelect / 32, kWords = 2 * kSelect, kPack = HELD ? 2 : 1, kPer = 2 * kPack;
    constexpr int kLog = (kSelect == 1024 ? 10 : 8) + kPack, kDigits = (31 + kLog) / kLog;
    static_assert(kPer * kSelect == 1 << kLog);
    extern __shared__ __align__(16) uint32_t s_key[];
    __shared__ __align__(8) uint32_t s_hist[kCopies + kDigits - 1][kWords];
    __shared__ int s_scan[32];
    __shared__ int s_digit, s_above, s_here;
    __shared__ int s_eq, s_last;              // read by the cluster's other CTAs
    __shared__ int s_holes[8], s_movers[8];   // every CTA's, written by them
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = blockIdx.x, ctas = gridDim.x;
    const int t = threadIdx.x, lane = t & 31, b = blockIdx.z;
    const size_t bh = static_cast<size_t>(b) * c.kv_heads + blockIdx.y;
    for (int i = t; i < (kCopies + kDigits - 1) * kWords; i += kSelect) (&s_hist[0][0])[i] = 0u;
    if (t == 0) s_last = -1;
    fer::dev::pdl_begin();
    __syncthreads();
    bool bad;
    const int n = c.length(b, &bad);
    if (bad && t == 0 && rank == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    const Head h = head_of(c, p, bh);
    if (p.fused && !p.late && t == 0 && rank == 0 && blockIdx.y == 0) p.new_lengths[b] = min(n, p.budget);
    if (n <= p.budget) {   // the same for the whole cluster
        copy_whole(h, n, rank * kSelect + t, ctas * kSelect);
        if (t == 0 && rank == 0) p.counts[bh] = 0;
        return;
    }
    const long long first = static_cast<long long>(p.seen[b]) - p.recent;
    const int each = fer::evict::slots_of_cta(n, ctas);
    const int lo = static_cast<int>(min(static_cast<long long>(n), static_cast<long long>(rank) * each));
    const int hi = min(n - lo, each) + lo;
    // slots a thread takes in a round: all of the CTA's in one round where keys are held
    const int run = HELD ? fer::evict::slots_of_thread(each, kSelect) : 32, round = run * kSelect;
    // this thread's slots of a round, `mine` on: fn(i, key)
    auto each_key = [&](int mine, auto fn) {
        if constexpr (HELD) {
#pragma unroll 2
            for (int i = 0; i < run; i += 4) {
                const int j = mine - lo + i;
                const uint4 v = *reinterpret_cast<const uint4*>(s_key + fer::evict::word_of(j));
                fn(i, v.x), fn(i + 1, v.y), fn(i + 2, v.z), fn(i + 3, v.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int j = min(mine + i, hi - 1);
                fn(i, key_of(h.w[j], h.pos[j], first));
            }
        }
    };
    auto meet = [&]() {
        if (ctas > 1) cluster.sync();
        else __syncthreads();
    };
    auto count_one = [&](uint32_t* hist, uint32_t bin) {
        if constexpr (HELD) atomicAdd(&hist[bin >> 1], bin & 1 ? 0x10000u : 1u);
        else atomicAdd(&hist[bin], 1u);
    };
    // keys, and the count of their first digit; kBatch loads in flight
    constexpr int kBatch = 8;
    for (int j0 = lo + t; j0 < hi; j0 += kBatch * kSelect) {
        float wt[kBatch];
        int pos[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int j = min(j0 + k * kSelect, hi - 1);
            wt[k] = h.w[j];
            pos[k] = h.pos[j];
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int j = j0 + k * kSelect;
            if (j >= hi) break;
            const uint32_t key = key_of(wt[k], pos[k], first);
            if constexpr (HELD) s_key[fer::evict::word_of(j - lo)] = key;
            count_one(s_hist[lane % kCopies], key >> (32 - kLog));
            if (j < p.budget) {
                if (h.nw != h.w) h.nw[j] = wt[k];
                if (h.np != h.pos) h.np[j] = pos[k];
            }
        }
    }
    uint32_t cut = 0u;
    int left = p.budget, equal = 0;   // slots to be found among the keys that begin like the cut, and how many those are
#pragma unroll
    for (int d = 0; d < kDigits; ++d) {
        const int above = 32 - d * kLog, shift = max(0, above - kLog), bins = 1 << (above - shift);
        uint32_t* const hist = s_hist[d == 0 ? 0 : kCopies + d - 1];
        if (d > 0) {
            const uint32_t mask = ~0u << above;   // the digits found so far
            for (int mine = lo + run * t; mine < hi; mine += round)
                each_key(mine, [&](int i, uint32_t key) {
                    if ((key & mask) == cut && mine + i < hi) count_one(hist, (key >> shift) & (bins - 1));
                });
        } else {
            __syncthreads();
            for (int i = t; i < kWords; i += kSelect) {
                uint32_t n0 = hist[i];
#pragma unroll
                for (int k = 1; k < kCopies; ++k) n0 += s_hist[k][i];
                hist[i] = n0;
            }
        }
        meet();
        // thread t has the kPer bins from kPer t on, counted from the top
        int count[kPer] = {};
        if (kPer * t < bins) {
            uint2 v[8];   // all in flight
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                v[r] = make_uint2(0u, 0u);
                if (r < ctas)
                    v[r] = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(hist, r) + (bins - kPer * (t + 1)) / kPack);
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if constexpr (HELD) {
                    count[0] += v[r].y >> 16, count[1] += v[r].y & 0xffffu;
                    count[2] += v[r].x >> 16, count[3] += v[r].x & 0xffffu;
                } else {
                    count[0] += v[r].y, count[1] += v[r].x;
                }
            }
        }
        int sum = 0, total;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += count[i];
        int before = block_scan<kWarps>(sum, s_scan, &total);
        if (before < left && left <= before + sum) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (before < left && left <= before + count[i]) {
                    s_digit = bins - 1 - (kPer * t + i);
                    s_above = before;
                    s_here = count[i];
                }
                before += count[i];
            }
        }
        __syncthreads();
        cut |= static_cast<uint32_t>(s_digit) << shift;
        left -= s_above;
        equal = s_here;
        __syncthreads();
        if (left == equal) break;   // every key that begins like the cut is kept
    }
    // of the slots whose key is the cut the first `left` are kept: those up to `last`
    int last = n;
    if (left < equal) {   // the same for the whole cluster
        auto word_of = [&](int mine) {
            uint32_t word = 0u;
            if (mine < hi) each_key(mine, [&](int i, uint32_t key) { word |= (key == cut ? 1u : 0u) << i; });
            return word & low_bits(min(run, hi - mine));
        };
        int before = 0, total;
        if (ctas > 1) {
            int mine = 0;
            for (int r0 = lo; r0 < hi; r0 += round) mine += __popc(word_of(r0 + run * t));
            block_scan<kWarps>(mine, s_scan, &total);
            if (t == 0) s_eq = total;
            cluster.sync();
            for (int r = 0; r < rank; ++r) before += *cluster.map_shared_rank(&s_eq, r);
        }
        for (int r0 = lo; r0 < hi; r0 += round) {
            uint32_t word = word_of(r0 + run * t);
            const int here = __popc(word);
            const int at = before + block_scan<kWarps>(here, s_scan, &total);
            if (at < left && left <= at + here) {   // the last one is this thread's
                for (int k = at + 1; k < left; ++k) word &= word - 1u;
                s_last = r0 + run * t + __ffs(word) - 1;
            }
            before += total;
        }
        meet();
        for (int r = 0; r < ctas; ++r) {
            const int v = *cluster.map_shared_rank(&s_last, r);
            if (v >= 0) last = v;
        }
    }
    // Freed slots before the budget and kept ones behind it: each thread has
    // its word of kept slots, and one scan of both counts, 16 bits each without
    // a sign (a round can have 32768), gives its places in the lists.
    auto low_half = [](int v) { return v & 0xffff; };
    auto high_half = [](int v) { return static_cast<int>(static_cast<uint32_t>(v) >> 16); };
    auto words = [&](int mine, uint32_t* hole, uint32_t* move) {
        uint32_t word = 0u;
        if (mine < hi) {
            each_key(mine, [&](int i, uint32_t key) { word |= (key >= cut ? 1u : 0u) << i; });
            if (last < mine + run - 1) {   // equal ones behind the last are not kept
                uint32_t equals = 0u;
                each_key(mine, [&](int i, uint32_t key) { equals |= (key == cut ? 1u : 0u) << i; });
                word &= ~equals | low_bits(last + 1 - mine);
            }
        }
        const uint32_t all = low_bits(min(run, hi - mine)), before = low_bits(p.budget - mine);
        word &= all;
        *hole = ~word & before & all;
        *move = word & ~before;
    };
    auto list = [&](int mine, uint32_t hole, uint32_t move, int h0, int m0) {
        for (; hole; hole &= hole - 1u, ++h0)
            if (h0 < p.cap) h.to[h0] = mine + __ffs(hole) - 1;
        for (; move; move &= move - 1u, ++m0)
            if (m0 < p.cap) h.from[m0] = mine + __ffs(move) - 1;
    };
    int holes = 0, movers = 0;    // of this CTA, or of its rounds so far
    int hole0 = 0, mover0 = 0;    // of the CTAs before
    auto earlier = [&]() {
        if (t < ctas) {
            *cluster.map_shared_rank(&s_holes[rank], t) = holes;
            *cluster.map_shared_rank(&s_movers[rank], t) = movers;
        }
        cluster.sync();   // the last: no CTA reads or writes another's shared memory behind it
        for (int r = 0; r < rank; ++r) hole0 += s_holes[r], mover0 += s_movers[r];
    };
    if constexpr (HELD) {   // one round
        static_assert(kMostKeys <= 32);
        const int mine = lo + run * t;
        uint32_t hole, move;
        int total;
        words(mine, &hole, &move);
        const int at = block_scan<kWarps>(__popc(hole) | __popc(move) << 16, s_scan, &total);
        holes = low_half(total);
        movers = high_half(total);
        if (ctas > 1) earlier();
        list(mine, hole, move, hole0 + low_half(at), mover0 + high_half(at));
    } else {
#pragma unroll 1
        for (int pass = ctas > 1 ? 0 : 1; pass < 2; ++pass) {
            for (int r0 = lo; r0 < hi; r0 += round) {
                const int mine = r0 + run * t;
                uint32_t hole, move;
                int total;
                words(mine, &hole, &move);
                const int at = block_scan<kWarps>(__popc(hole) | __popc(move) << 16, s_scan, &total);
                if (pass == 1) list(mine, hole, move, hole0 + holes + low_half(at), mover0 + movers + high_half(at));
                holes += low_half(total);
                movers += high_half(total);
            }
            if (pass == 0) {
                earlier();
                holes = movers = 0;
            }
        }
    }
    // all alike, unless the arrays changed meanwhile
    if (!HELD || !p.fused) {
        if (rank == ctas - 1 && t == 0) p.counts[bh] = min(mover0 + movers, min(hole0 + holes, p.cap));
        return;
    }
    // the cluster's warps share the moves out among them
    if (ctas > 1) {
        holes = movers = 0;
        for (int r = 0; r < ctas; ++r) holes += s_holes[r], movers += s_movers[r];
    }
    const int moved = min(movers, min(holes, p.cap));
    const int share = max(1, min(32, (moved - 1) / (kWarps * ctas) + 1));
    meet();   // the lists are written
    const int32_t* const row = c.table + static_cast<size_t>(b) * c.max_pages;
    for (int i0 = (rank * kWarps + (t >> 5)) * share; i0 < moved; i0 += kWarps * ctas * share) {
        const bool mine = lane < share && i0 + lane < moved;
        const int from = mine ? h.from[i0 + lane] : 0, to = mine ? h.to[i0 + lane] : 0;
        move_rows<D, 4>(c, p, h, blockIdx.y, mine, from, to, row[from >> c.shift], row[to >> c.shift]);
    }
}

// grid (move tiles, kv_heads, batch), a warp kWarpMoves moves
template <int D>
__global__ void __launch_bounds__(kMove) evict_move(const Paged c, const EvictParams p, const bool lengths) {
    fer::dev::pdl_begin();
    const int b = blockIdx.z, hk = blockIdx.y, lane = threadIdx.x & 31;
    const size_t bh = static_cast<size_t>(b) * c.kv_heads + hk;
    if (lengths && hk == 0 && blockIdx.x == 0 && threadIdx.x == 0) {   // the only reader of this length in the launch
        bool bad;
        p.new_lengths[b] = min(c.length(b, &bad), p.budget);
    }
    const int moved = p.counts[bh];
    const int i0 = (blockIdx.x * (kMove / 32) + (threadIdx.x >> 5)) * kWarpMoves, i = i0 + lane;
    if (i0 >= moved) return;
    const bool mine = lane < kWarpMoves && i < moved;
    const Head h = head_of(c, p, bh);
    const int from = mine ? h.from[i] : 0, to = mine ? h.to[i] : 0;
    const int32_t* const row = c.table + static_cast<size_t>(b) * c.max_pages;
    move_rows<D, 8>(c, p, h, hk, mine, from, to, row[from >> c.shift], row[to >> c.shift]);
}

__global__ void __launch_bounds__(kMove) evict_lengths(const Paged c, const EvictParams p, const int batch) {
    fer::dev::pdl_begin();
    const int b = blockIdx.x * kMove + threadIdx.x;
    bool bad;
    if (b < batch) p.new_lengths[b] = min(c.length(b, &bad), p.budget);
}

int most_moves(int max_slots, int budget) {
    const int behind = max_slots - budget;
    return behind < budget ? behind : budget;
}

size_t up16(size_t v) { return (v + 15) & ~size_t(15); }

// As launch_pdl, in clusters of `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t s,
                           Args&&... args) {
    if (cluster == 1) return fer::host::launch_pdl(kern, grid, block, smem, s, std::forward<Args>(args)...);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = fer::host::pdl_enabled() ? 2 : 1;
    fer_pdl_note_launch();   // the kernel triggers its dependents either way
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

template <int D, int KEYS>
cudaError_t small(const Paged& c, const EvictParams& p, int batch, cudaStream_t s) {
    // two heads a CTA, up to eight CTAs a sequence
    unsigned ctas = 1;
    while (ctas < 8 && 4 * ctas <= static_cast<unsigned>(c.kv_heads)) ctas *= 2;
    const int warps = (c.kv_heads + ctas - 1) / ctas < 8 ? (c.kv_heads + ctas - 1) / ctas : 8;
    const unsigned cluster = p.new_lengths == c.lengths ? ctas : 1;
    return launch_cluster(evict_small<D, KEYS>, dim3(ctas, batch), dim3(32 * warps), 0, cluster, s, c, p);
}

template <int D, bool HELD, int THREADS>
cudaError_t select(const Paged& c, const EvictParams& p, unsigned ctas, int batch, cudaStream_t s) {
    const auto kernel = evict_select<D, HELD, THREADS>;
    const int each = fer::evict::slots_of_cta(c.max_slots(), static_cast<int>(ctas));
    const size_t smem = HELD ? sizeof(uint32_t) * fer::evict::words_of_cta(each, THREADS) : 0;
    if (HELD) {
        static std::atomic<bool> set[fer::host::kMaxDevices];
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= fer::host::kMaxDevices || !set[dev].load(std::memory_order_relaxed)) {
            constexpr int most = sizeof(uint32_t) * fer::evict::words_of_cta(kMostKeys * THREADS, THREADS);
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
            if (e != cudaSuccess) return e;
            if (dev < fer::host::kMaxDevices) set[dev].store(true, std::memory_order_relaxed);
        }
    }
    return launch_cluster(kernel, dim3(ctas, c.kv_heads, batch), dim3(THREADS), smem, ctas, s, c, p);
}

template <int D>
cudaError_t run(const Paged& c, EvictParams& p, int batch, cudaStream_t s) {
    cudaError_t e;
    const int max_slots = c.max_slots();
    const bool few = max_slots <= kSmall;
    if (few) {
        p.fused = p.cap <= kFusedMoves;
        e = max_slots <= 256   ? small<D, 8>(c, p, batch, s)
            : max_slots <= 512 ? small<D, 16>(c, p, batch, s)
            : max_slots <= 768 ? small<D, 24>(c, p, batch, s)
                               : small<D, 32>(c, p, batch, s);
        if (e != cudaSuccess || p.fused) return e;
    } else {
        // As many CTAs a head as its keys need; more where SMs would be left over, a CTA at least 4096 slots
        // (32 heads of 32768 slots: 20 us with one CTA a head, 18 with four). Eight only for up to eight heads:
        // clusters of eight do not fill all SMs (16 heads of 32768 slots: 32 us in all with four, 44 with eight).
        const long long heads = static_cast<long long>(c.kv_heads) * batch;
        unsigned ctas = 1;
        while (ctas < 8 && static_cast<long long>(ctas) * kMostKeys * kSelect < max_slots) ctas *= 2;
        while (ctas < 4 && 2 * ctas * heads <= 148 && ctas * 4096ll < max_slots) ctas *= 2;
        if (ctas == 4 && heads <= 8 && 4 * 4096 < max_slots) ctas = 8;
        // In several waves the moves of one head overlap the selection of others (512 heads of 8192 slots cut to
        // 4096, rows of 64: 202 us in two kernels, 152 in one); in one wave they gain nothing (32 heads: 32.2 and
        // 32.0) or, with few CTAs, are slower (1 head of 8192: 23.8 and 32.4).
        const bool held = max_slots <= static_cast<long long>(ctas) * kMostKeys * kSelect;
        p.fused = held && ctas * heads >= kFuseCtas;
        p.late = p.new_lengths == c.lengths;
        // More heads than SMs, and short ones: several small CTAs an SM hide one another's latencies (1344 heads of
        // 1560 slots cut to 542: 121 us with 1024 threads, 77 with 256; 320 of 8000 to 7990: 36 and 26). With many
        // moves a head large CTAs in more waves overlap better (512 of 8192 to 4096: 153 and 174).
        const bool small_ctas = heads > 148 && max_slots <= kMostKeys * kSelectFew && p.cap <= 2048;
        e = !held        ? select<D, false, kSelect>(c, p, ctas, batch, s)
            : small_ctas ? select<D, true, kSelectFew>(c, p, ctas, batch, s)
                         : select<D, true, kSelect>(c, p, ctas, batch, s);
        if (e != cudaSuccess || (p.fused && !p.late)) return e;
        if (p.fused)
            return fer::host::launch_pdl(evict_lengths, dim3((batch + kMove - 1) / kMove), dim3(kMove), 0, s, c, p, batch);
    }
    constexpr int kTile = kMove / 32 * kWarpMoves;
    const dim3 grid((p.cap + kTile - 1) / kTile + (p.cap == 0), c.kv_heads, batch);
    return fer::host::launch_pdl(evict_move<D>, grid, dim3(kMove), 0, s, c, p, !few);
}

}  // namespace

extern "C" size_t fer_paged_evict_workspace_bytes(int batch, int kv_heads, int max_slots, int budget) {
    if (batch <= 0 || kv_heads <= 0 || budget <= 0) return 0;
    const size_t bh = static_cast<size_t>(batch) * kv_heads;
    const int cap = most_moves(max_slots, budget);
    return up16(bh * 4) + (cap > 0 ? 2 * up16(bh * cap * 4) : 0);
}

extern "C" cudaError_t fer_paged_evict(const fer_paged_view_t* cache, const fer_paged_evict_args_t* a, uint32_t* err,
                                       cudaStream_t s) {
    Paged c{};
    const cudaError_t ce = fer::host::paged_params(cache, &c);
    if (ce != cudaSuccess) return ce;
    if (!a || a->budget < 1 || a->recent < 0 || a->recent > a->budget || !a->weights || !a->positions || !a->seen ||
        !a->new_lengths || !a->new_weights || !a->new_positions)
        return cudaErrorInvalidValue;
    if (!fer::host::words_aligned({a->weights, a->positions, a->seen, a->new_lengths, a->new_weights, a->new_positions}))
        return cudaErrorInvalidValue;
    if (c.kv_heads > 65535 || cache->batch > 65535) return cudaErrorNotSupported;
    const int max_slots = c.max_slots();
    const size_t need = fer_paged_evict_workspace_bytes(cache->batch, c.kv_heads, max_slots, a->budget);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need)
        return cudaErrorInvalidValue;
    EvictParams p{};
    p.budget = a->budget;
    p.recent = a->recent;
    p.cap = most_moves(max_slots, a->budget) > 0 ? most_moves(max_slots, a->budget) : 0;
    p.weights = a->weights;
    p.positions = a->positions;
    p.seen = a->seen;
    p.new_lengths = a->new_lengths;
    p.new_weights = a->new_weights;
    p.new_positions = a->new_positions;
    const size_t bh = static_cast<size_t>(cache->batch) * c.kv_heads;
    char* w = static_cast<char*>(a->workspace);
    p.counts = reinterpret_cast<int32_t*>(w);
    w += up16(bh * 4);
    p.to = reinterpret_cast<int32_t*>(w);
    w += up16(bh * p.cap * 4);
    p.from = reinterpret_cast<int32_t*>(w);
    p.err = err;
    cudaError_t e;
    switch (c.head_dim) {
        case 64: e = run<64>(c, p, cache->batch, s); break;
        case 128: e = run<128>(c, p, cache->batch, s); break;
        default: e = run<256>(c, p, cache->batch, s); break;
    }
    return e;
}
