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
// Up to 1024 slots (evict_small): a warp a head with its keys in registers,
// lane-strided, finds the cut bit by bit: at most 32 counts, no shared memory
// and no barrier, and it stops as soon as a cut leaves exactly the budget.
// What a lane frees, keeps and moves are then 32-bit masks, and only the key
// registers that hold such a slot in some lane cost a ballot. A sequence's
// heads share a cluster, so that its length can be replaced once all have
// read it. When a head can have at most 32 moves (a cache that is cut back every few
// tokens) the warp also makes them, and one launch does it all.
//
// Above (evict_select): a CTA a head, from 48K slots on a cluster of 2 to 8,
// with the keys in shared memory, and three digits of 11, 11 and 10 bits counted there; the
// other CTAs' counts are read through distributed shared memory. Beyond 8 x
// 48K slots the keys are made again for every pass.
//
// The moves (evict_move): a warp resolves 32 moves at once, a lane each, then
// copies their rows with kAhead 16-byte loads a lane in flight.
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
constexpr int kSelect = 1024;                // threads of a selecting CTA
constexpr int kWarps = kSelect / 32;
constexpr int kMostKeys = 48 * 1024;         // keys a CTA holds in shared memory
constexpr int kBins = 2048;
constexpr int kMove = 256;
constexpr int kFusedMoves = 32;

struct EvictParams {
    int budget, recent, cap;     // cap: moves a (sequence, key head) can have
    int fused;                   // the selecting warp moves rows
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
template <int D>
__device__ __forceinline__ void move_rows(const Paged& c, const EvictParams& p, const Head& h, int b, int hk,
                                          bool mine, int from, int to) {
    constexpr int kPieces = D / 8, kRows = 32 / kPieces, kAhead = 8;   // lanes a row, rows at once
    const int lane = threadIdx.x & 31, piece = lane % kPieces;
    unsigned long long src = 0, dst = 0;
    bool good = false;
    if (mine) {
        const int pf = c.page(b, from), pt = c.page(b, to);
        h.nw[to] = h.w[from];
        h.np[to] = h.pos[from];
        good = pf >= 0 && pt >= 0;
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

// grid (CTAs a sequence, batch), a cluster a sequence and a warp a head, for
// max_slots <= 32 * KEYS. Slot 32 i + lane is key i of that lane.
template <int D, int KEYS>
__global__ void __launch_bounds__(256) evict_small(const Paged c, const EvictParams p) {
    __shared__ int s_to[8][kFusedMoves], s_from[8][kFusedMoves];
    const cg::cluster_group cluster = cg::this_cluster();
    const int b = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int warps = blockDim.x >> 5, step = warps * gridDim.x;
    fer::dev::pdl_begin();
    bool bad;
    const int n = c.length(b, &bad);
    if (bad && threadIdx.x == 0 && blockIdx.x == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    const long long first = static_cast<long long>(p.seen[b]) - p.recent;
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
        for (int bit = 31; bit >= 0 && above != p.budget; --bit) {
            const uint32_t next = cut | 1u << bit;
            int m = 0;
#pragma unroll
            for (int i = 0; i < KEYS; ++i) m += key[i] >= next ? 1 : 0;   // next > 0: slots behind n do not count
            m = __reduce_add_sync(kAll, m);
            if (m >= p.budget) cut = next, above = m;
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
            move_rows<D>(c, p, h, b, hk, lane < moved, lane < moved ? from[lane] : 0, lane < moved ? to[lane] : 0);
            __syncwarp();
        } else if (lane == 0) {
            p.counts[bh] = moved;
        }
    }
    cluster.sync();   // every head has read the length
    if (blockIdx.x == 0 && threadIdx.x == 0) p.new_lengths[b] = min(n, p.budget);
}

// Exclusive prefix sum over the block, and the total.
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
// hi), warp w of it the run [a, z) of those: runs are in slot order.
__global__ void __launch_bounds__(kSelect, 1) evict_select(const Paged c, const EvictParams p, const int room) {
    extern __shared__ uint32_t s_key[];       // [room], the CTA's keys where they fit
    __shared__ __align__(8) int s_hist[3][kBins];
    __shared__ int s_scan[32];
    __shared__ int s_digit, s_above, s_here;
    __shared__ int s_eq, s_last;              // read by the cluster's other CTAs, as are the next two
    __shared__ int s_holes, s_movers;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = blockIdx.x, ctas = gridDim.x;
    const int t = threadIdx.x, lane = t & 31, w = t >> 5, b = blockIdx.z;
    const size_t bh = static_cast<size_t>(b) * c.kv_heads + blockIdx.y;
    fer::dev::pdl_begin();
    bool bad;
    const int n = c.length(b, &bad);
    if (bad && t == 0 && rank == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    const Head h = head_of(c, p, bh);
    if (n <= p.budget) {   // the same for the whole cluster
        copy_whole(h, n, rank * kSelect + t, ctas * kSelect);
        if (t == 0 && rank == 0) p.counts[bh] = 0;
        return;
    }
    const long long first = static_cast<long long>(p.seen[b]) - p.recent;
    const int each = ((n - 1) / ctas + 1 + 127) & ~127;
    const int lo = static_cast<int>(min(static_cast<long long>(n), static_cast<long long>(rank) * each));
    const int hi = min(n - lo, each) + lo;
    const bool held = each <= room;
    const int run = ((hi - lo + kWarps - 1) / kWarps + 31) & ~31;
    const int a = min(hi, lo + w * run), z = min(hi, a + run);
    auto key_at = [&](int j) { return held ? s_key[j - lo] : key_of(h.w[j], h.pos[j], first); };
    auto meet = [&]() {
        if (ctas > 1) cluster.sync();
        else __syncthreads();
    };
    for (int i = t; i < 3 * kBins; i += kSelect) (&s_hist[0][0])[i] = 0;
    if (t == 0) s_last = -1;
    __syncthreads();
    // keys, and the count of their first digit; kBatch loads in flight
    constexpr int kBatch = 4;
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
            if (held) s_key[j - lo] = key;
            atomicAdd(&s_hist[0][key >> 21], 1);
            if (j < p.budget) {
                if (h.nw != h.w) h.nw[j] = wt[k];
                if (h.np != h.pos) h.np[j] = pos[k];
            }
        }
    }
    uint32_t cut = 0u;
    int left = p.budget, equal = 0;   // slots to be found among the keys that begin like the cut, and how many those are
#pragma unroll
    for (int d = 0; d < 3; ++d) {
        const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bins = d == 2 ? 1024 : 2048;
        if (d > 0) {
            const uint32_t mask = d == 1 ? 0xffe00000u : 0xfffffc00u;   // the digits found so far
#pragma unroll 4
            for (int j = lo + t; j < hi; j += kSelect) {
                const uint32_t key = key_at(j);
                if ((key & mask) == cut) atomicAdd(&s_hist[d][(key >> shift) & (bins - 1)], 1);
            }
        }
        meet();
        // thread t has the kPer bins from kPer t on, counted from the top
        constexpr int kPer = kBins / kSelect;
        static_assert(kPer == 2);
        int count[kPer] = {}, sum = 0;
        if (kPer * t < bins) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r >= ctas) break;
                const int2 v = *reinterpret_cast<const int2*>(cluster.map_shared_rank(&s_hist[d][0], r) + bins - kPer * (t + 1));
                count[0] += v.y, count[1] += v.x;
            }
        }
        sum = count[0] + count[1];
        int total;
        int before = block_scan(sum, s_scan, &total);
        if (before < left && left <= before + sum) {
            const bool second = left > before + count[0];
            s_digit = bins - 1 - (kPer * t + (second ? 1 : 0));
            s_above = before + (second ? count[0] : 0);
            s_here = second ? count[1] : count[0];
        }
        __syncthreads();
        cut |= static_cast<uint32_t>(s_digit) << shift;
        left -= s_above;
        equal = s_here;
        __syncthreads();
    }
    // of the slots whose key is the cut the first `left` are kept: those up to `last`
    int last = n;
    if (left < equal) {   // the same for the whole cluster
        int eq = 0;
        for (int j = a + lane; j < z; j += 32) eq += key_at(j) == cut ? 1 : 0;
        eq = __reduce_add_sync(kAll, eq);
        int total;
        int before = __shfl_sync(kAll, block_scan(lane == 0 ? eq : 0, s_scan, &total), 0);
        if (t == 0) s_eq = total;
        meet();
        for (int r = 0; r < rank; ++r) before += *cluster.map_shared_rank(&s_eq, r);
        if (before < left && left <= before + eq) {   // the last one lies in this warp's run
            for (int j0 = a; j0 < z; j0 += 32) {
                const uint32_t row = __ballot_sync(kAll, j0 + lane < z && key_at(min(j0 + lane, z - 1)) == cut);
                if (before + __popc(row) >= left) {
                    if ((row >> lane & 1u) && before + __popc(row & low_bits(lane)) + 1 == left) s_last = j0 + lane;
                    break;
                }
                before += __popc(row);
            }
        }
        meet();
        for (int r = 0; r < ctas; ++r) {
            const int v = *cluster.map_shared_rank(&s_last, r);
            if (v >= 0) last = v;
        }
    }
    auto kept_at = [&](int j) {
        const uint32_t key = key_at(j);
        return key > cut || (key == cut && j <= last);
    };
    // freed slots before the budget and kept ones behind it, counted, then listed
    int holes = 0, movers = 0;
#pragma unroll 4
    for (int j = a + lane; j < z; j += 32) {
        const bool kept = kept_at(j);
        holes += !kept && j < p.budget ? 1 : 0;
        movers += kept && j >= p.budget ? 1 : 0;
    }
    holes = __reduce_add_sync(kAll, holes);
    movers = __reduce_add_sync(kAll, movers);
    int all_holes, all_movers;
    int hole0 = __shfl_sync(kAll, block_scan(lane == 0 ? holes : 0, s_scan, &all_holes), 0);
    int mover0 = __shfl_sync(kAll, block_scan(lane == 0 ? movers : 0, s_scan, &all_movers), 0);
    if (t == 0) s_holes = all_holes, s_movers = all_movers;
    meet();
    int before_h = 0, before_m = 0;
    for (int r = 0; r < rank; ++r) {
        before_h += *cluster.map_shared_rank(&s_holes, r);
        before_m += *cluster.map_shared_rank(&s_movers, r);
    }
    hole0 += before_h;
    mover0 += before_m;
#pragma unroll 4
    for (int j0 = a; j0 < z; j0 += 32) {
        const int j = j0 + lane;
        const bool kept = j < z && kept_at(j), front = j < p.budget;
        const uint32_t hole = __ballot_sync(kAll, j < z && !kept && front), move = __ballot_sync(kAll, kept && !front);
        const int nh = hole0 + __popc(hole & low_bits(lane)), nm = mover0 + __popc(move & low_bits(lane));
        if ((hole >> lane & 1u) && nh < p.cap) h.to[nh] = j;
        if ((move >> lane & 1u) && nm < p.cap) h.from[nm] = j;
        hole0 += __popc(hole);
        mover0 += __popc(move);
    }
    // all alike, unless the arrays changed meanwhile
    if (rank == ctas - 1 && t == 0)
        p.counts[bh] = min(before_m + all_movers, min(before_h + all_holes, p.cap));
    if (ctas > 1) cluster.sync();   // no CTA leaves while another may read its shared memory
}

// grid (move tiles, kv_heads, batch), a warp 32 moves
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
    const int i = (blockIdx.x * (kMove / 32) + (threadIdx.x >> 5)) * 32 + lane;
    if (i - lane >= moved) return;
    const Head h = head_of(c, p, bh);
    move_rows<D>(c, p, h, b, hk, i < moved, i < moved ? h.from[i] : 0, i < moved ? h.to[i] : 0);
}

int most_moves(int max_slots, int budget) {
    const int behind = max_slots - budget;
    return behind < budget ? behind : budget;
}

size_t up16(size_t v) { return (v + 15) & ~size_t(15); }

constexpr int kDevices = 64;

cudaError_t launch_cluster(const void* kernel, dim3 grid, int threads, size_t smem, unsigned cluster, cudaStream_t s,
                           void** args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
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
    fer_pdl_note_launch();
    return cudaLaunchKernelExC(&cfg, kernel, args);
}

template <int D>
const void* small_kernel(int max_slots) {
    const void* k[] = {reinterpret_cast<const void*>(evict_small<D, 8>), reinterpret_cast<const void*>(evict_small<D, 16>),
                       reinterpret_cast<const void*>(evict_small<D, 24>), reinterpret_cast<const void*>(evict_small<D, 32>)};
    return k[(max_slots - 1) / 256];
}

template <int D>
cudaError_t run(const Paged& c, EvictParams& p, int batch, cudaStream_t s) {
    cudaError_t e;
    const int max_slots = c.max_slots();
    const bool small = max_slots <= kSmall;
    if (small) {
        p.fused = p.cap <= kFusedMoves;
        // two heads a CTA, up to eight CTAs a sequence
        unsigned ctas = 1;
        while (ctas < 8 && 4 * ctas <= static_cast<unsigned>(c.kv_heads)) ctas *= 2;
        const int warps = (c.kv_heads + ctas - 1) / ctas < 8 ? (c.kv_heads + ctas - 1) / ctas : 8;
        Paged view = c;
        void* args[] = {&view, &p};
        e = launch_cluster(small_kernel<D>(max_slots), dim3(ctas, batch), 32 * warps, 0, ctas, s, args);
        if (e != cudaSuccess || p.fused) return e;
    } else {
        // no more CTAs a head than its keys need: a step of a cluster (barrier, remote counts) takes about 2 us,
        // which is what one SM takes to read 10,000 more slots
        unsigned ctas = 1;
        while (ctas < 8 && static_cast<long long>(ctas) * kMostKeys < max_slots) ctas *= 2;
        long long room = ((max_slots - 1) / static_cast<int>(ctas) + 1 + 127) & ~127;
        if (room > kMostKeys) room = 0;
        int keys = static_cast<int>(room);
        static std::atomic<bool> set[kDevices];
        int dev = 0;
        e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= kDevices || !set[dev].load(std::memory_order_relaxed)) {
            e = cudaFuncSetAttribute(evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kMostKeys);
            if (e != cudaSuccess) return e;
            if (dev < kDevices) set[dev].store(true, std::memory_order_relaxed);
        }
        Paged view = c;
        void* args[] = {&view, &p, &keys};
        e = launch_cluster(reinterpret_cast<const void*>(evict_select), dim3(ctas, c.kv_heads, batch), kSelect,
                           4 * static_cast<size_t>(keys), ctas, s, args);
        if (e != cudaSuccess) return e;
    }
    const dim3 grid((p.cap + kMove - 1) / kMove + (p.cap == 0), c.kv_heads, batch);
    return fer::host::launch_pdl(evict_move<D>, grid, dim3(kMove), 0, s, c, p, !small);
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
    return e != cudaSuccess ? e : cudaGetLastError();
}
