// Attention of one new token per sequence over a paged key-value cache.
//
// For a query head h with key head h / group: s_j = scale q.k_j over the held
// slots j, out = sum_j p_j v_j with p = exp(s - lse). Every key and value is
// read once for all heads of a group and takes 4 flops a head and element, so
// the pass is bound by HBM reads of the cache.
//
// Split. A sequence's slots are cut into chunks at fixed places; a unit of
// work is (sequence, key head, block of 8 or 16 query heads, chunk). Every CTA
// counts the units and their cost from the lengths and takes a contiguous run
// of equal cost, so ragged batches and tables much wider than the lengths are
// shared out evenly without the host knowing the lengths; where every unit
// there can be has a CTA of its own, its index is the unit. A unit's maximum m,
// l = sum 2^(s - m) and o = sum 2^(s - m) v go to the workspace in f32 (or,
// with one chunk, the result to the output), and a second kernel joins a head's
// chunks: 8 or 16 partial sums of every 8th or 16th chunk each, then those in
// order. How many depends on the table's width, and how many chunks share a
// maximum on head_dim. Which CTA took a unit does not change its arithmetic:
// results are the same run to run and for any batch.
//
// Inside a unit a warp loads rounds of 64 slots by tensor copies of page rows
// into a ring, running on into the next units, and four warps compute. In a
// round each of them takes 16 slots' scores for all heads, S^T = K Q^T; they
// agree on the maxima, exchange their probabilities through shared memory as
// ready operand fragments, and each then adds a quarter of the dims, O^T = V^T
// P, over all 64 slots. So an output stays in one warp (no sums to be joined at
// a unit's end) and takes few registers, and several CTAs share an SM and hide
// one another's latencies. Products are 16-bit tensor-core tiles with f32
// accumulation: with slots or dims as rows the 8 columns are the heads, so a
// group of up to 8 heads wastes nothing it would have to read. (A group of up
// to 16 heads is 1/8 of the 128 rows a tcgen05 tile has, and the tiles here run
// at a few per cent of the tensor pipe. Larger groups read their pages once
// more, from L2, for every 16 heads: 64 heads over one key head, 64 sequences
// of up to 2048 slots, take 47 us, ten times their bytes at the copy rate;
// there heads as a tcgen05 tile's rows would fit.)
// P is kept as the sum of two 16-bit numbers, so it has 16 bits or more:
// rounding it once would have added half of the output's own rounding error.
//
// Measured (HBM copy 6538 GB/s): 131071 slots x 8 key heads of 128 for 64
// heads 91 to 92.5 us, 5.8 TB/s; 33 sequences of 0 to 8192 slots with weights 115
// us (86 us at the copy rate); 64 sequences of 1 to 1024 slots x 16 heads of 64
// 32 to 33.2 us (20.6): 3.5 us pass until the first rows arrive, CTAs end between 18
// and 29 us as they have a unit more or less, and 5 us go to the joining.
//
// Scores are kept in base-2 units (scale * log2 e folded into one factor).
// When weights are wanted they go to the workspace as well, and the second
// kernel adds 2^(s - lse) of a group's heads, in head order.
//
// A chunk whose scores are all -inf has l = 0 and counts as empty (m = 0 in
// its exponents, so no inf - inf); l = 0 over all chunks gives zeros.
#include "paged.cuh"
#include "pdl.cuh"
#include "tmap.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>

namespace {

using fer::dev::Paged;
constexpr int kWarps = 4;                        // that compute; one more loads
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kRound = 16 * kWarps;  // slots a round
constexpr int kTiles = 148 * 16;     // CTAs that add weights, at least where there are that many tiles
constexpr int kManyHeads = 148 * 4;  // heads whose joining fills the GPU with a CTA each
constexpr int kSegments = 128;       // entries of the unit table in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMostScale = 2.0e38f;   // times log2 e it is still finite
constexpr float kLn2 = 0.6931471805599453f;

// Slots a chunk: a function of the table's width alone, so that a sequence's
// results do not depend on the batch. Short chunks share the work out more
// evenly, long ones write fewer parts: 2 x 40003 slots with weights take 39.2 us
// in chunks of 512 and 36.6 of 256, 131071 slots 91.1 of 512 and 97.5 of 256.
__host__ __device__ inline int chunk_of(int max_slots) { return max_slots > 65536 ? 512 : 256; }

struct AttnParams {
    const void* q;
    void* out;
    size_t qs, os;
    int n_seq, heads, group, blocks, chunks;   // blocks: head blocks a key head
    int chunk_log2;
    int direct;          // every unit there can be has a CTA of its own
    __device__ __forceinline__ int chunk() const { return 1 << chunk_log2; }
    __device__ __forceinline__ int chunks_of(int len) const { return (len + chunk() - 1) >> chunk_log2; }
    float scale2;        // scale * log2 e
    float* lse;
    float* weights;
    float* part_ml;      // [n_seq * heads][chunks][2]
    float* part_o;       // [n_seq * heads][chunks][head_dim]
    float* scores;       // [n_seq * heads][max_slots], with weights
    uint32_t* err;
};

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// Tensor copy of a box of rows of one page: 64 dims from x, rows from r.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int r, int head, int page,
                                         uint32_t bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::
            "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r), "r"(head), "r"(page), "r"(bar), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
// Barrier of the computing warps.
__device__ __forceinline__ void meet_warps() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }
// Transposes an 8 x 8 tile of 16-bit elements spread over the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && __is_same(T, __half))
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (x, y), not negative, as two 16-bit numbers each: cut off, and what that
// leaves. Both parts are at least the smallest positive number, so that an
// infinite value gives an infinite product and not 0 x inf; NaN stays NaN.
// f16 parts are of 2^14 x, which keeps 2^-38 and up; the sum over v is scaled
// back at a unit's end.
template <typename T>
constexpr float kScaleP = __is_same(T, __half) ? 16384.0f : 1.0f;
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (__is_same(T, __half)) {
        x *= kScaleP<T>;
        y *= kScaleP<T>;
        float hx, hy;
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
            : "=f"(hx), "=f"(hy)
            : "r"(hi));
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(y - hy), "f"(x - hx));
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x00010001u));
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x00010001u));
    } else {
        const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
        hi = __byte_perm(ux, uy, 0x7632);
        const float rx = x - __uint_as_float(ux & 0xffff0000u), ry = y - __uint_as_float(uy & 0xffff0000u);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(ry), "f"(rx));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x00800080u));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x00800080u));
    }
}

// How a head_dim is cut: rounds in flight, CTAs an SM. A round's rows lie in
// bands of 64 dims, each as the copies write it: piece c (16 bytes) of row r
// at r * 128 + ((c ^ (r % 8)) * 16), so eight rows' pieces of one column are
// in different banks.
template <int D> struct Cut {
    static constexpr int kStages = D == 128 ? 2 : 3;
    static constexpr int kCtas = D == 64 ? 4 : D == 128 ? 3 : 1;
    static constexpr int kBand = kRound * 128;
    static constexpr int kHalf = D / 64 * kBand;             // keys; the values follow
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kSmem = kStages * kStage + 1024;    // bands start at 1024 bytes
    // Byte of piece c of row r in a half of a stage.
    static __device__ __forceinline__ uint32_t at(int r, int c) {
        return (c >> 3) * kBand + r * 128 + (((c ^ r) & 7) << 4);
    }
};

// What a unit costs, in rounds: its rounds, and kUnitCost more for its
// beginning and its end.
constexpr int kUnitCost = 1;
__host__ __device__ inline int rounds_of(int n) { return (n + kRound - 1) / kRound; }

// The units and the cost before every segment of sequences; in shared memory.
struct Units {
    const int* units;
    const int* cost;   // both [segments], ascending
    int segments, seg;

    // The last segment that starts at or before v.
    __device__ __forceinline__ int find(const int* list, int v) const {
        int lo = 0, hi = segments;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (list[mid] <= v) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};

// One sequence's units: head blocks, chunks of each, and the cost of a block.
struct Seq {
    int len, chunks, heads;
    __device__ __forceinline__ Seq(const Paged& c, const AttnParams& p, int b) {
        bool bad;
        len = c.length(b, &bad);
        chunks = p.chunks_of(len);
        heads = c.kv_heads * p.blocks;
    }
    __device__ __forceinline__ int units() const { return chunks * heads; }
    __device__ __forceinline__ int block_cost() const { return rounds_of(len) + chunks * kUnitCost; }
    __device__ __forceinline__ int cost() const { return block_cost() * heads; }
};

// The first unit whose cost begins at or behind x.
__device__ __forceinline__ int unit_at(const Paged& c, const AttnParams& p, const Units& t, int x) {
    const int s = t.find(t.cost, x);
    int u = t.units[s];
    x -= t.cost[s];
    for (int b = s * t.seg; b < min(p.n_seq, (s + 1) * t.seg); ++b) {
        const Seq q(c, p, b);
        if (x < q.cost()) {
            const int block = x / q.block_cost(), rest = x - block * q.block_cost();
            const int each = rounds_of(p.chunk()) + kUnitCost;
            return u + block * q.chunks + min((rest + each - 1) / each, q.chunks);
        }
        x -= q.cost();
        u += q.units();
    }
    return u;
}

// One unit.
struct Unit {
    int b, hk, blk, chunk, chunks, n;   // n: slots
};

__device__ __forceinline__ Unit find_unit(const Paged& c, const AttnParams& p, const Units& t, int u) {
    const int s = t.find(t.units, u);
    int r = u - t.units[s];
    int b = s * t.seg;
    Seq q(c, p, b);
    while (r >= q.units() && b + 1 < p.n_seq) {
        r -= q.units();
        q = Seq(c, p, ++b);
    }
    Unit x;
    x.b = b;
    x.chunks = q.chunks;
    const int hb = q.chunks > 0 ? r / q.chunks : 0;
    x.chunk = r - hb * q.chunks;
    x.hk = hb / p.blocks;
    x.blk = hb - x.hk * p.blocks;
    x.n = min(p.chunk(), q.len - (x.chunk << p.chunk_log2));
    return x;
}

// The units of a run, found 32 at a time, one a lane, and handed to the whole
// warp one by one.
struct UnitRun {
    int from = -1;   // unit of lane 0
    Unit x{};
    __device__ __forceinline__ Unit get(const Paged& c, const AttnParams& p, const Units& t, int u, int last) {
        if (from < 0 || u >= from + 32) {
            from = u;
            x = find_unit(c, p, t, min(u + static_cast<int>(threadIdx.x & 31), last));
        }
        const int i = u - from;
        Unit y;
        y.b = __shfl_sync(0xffffffffu, x.b, i);
        y.hk = __shfl_sync(0xffffffffu, x.hk, i);
        y.blk = __shfl_sync(0xffffffffu, x.blk, i);
        y.chunk = __shfl_sync(0xffffffffu, x.chunk, i);
        y.chunks = __shfl_sync(0xffffffffu, x.chunks, i);
        y.n = __shfl_sync(0xffffffffu, x.n, i);
        return y;
    }
};

// Page ids of a unit's chunk (up to 64 pages) as the table has them: lane i
// holds those of its i-th and (i + 32)-th page, -1 behind the last. They are
// checked where they are used, so that a load for a later unit stays in
// flight. k0: first slot of the chunk.
struct ChunkPages {
    int a, b;
    __device__ __forceinline__ int of(const Paged& c, int k0, int slot) const {   // a slot of the chunk
        const int i = ((k0 + slot) >> c.shift) - (k0 >> c.shift);
        const int x = __shfl_sync(0xffffffffu, a, i & 31), y = __shfl_sync(0xffffffffu, b, i & 31);
        return i < 32 ? x : y;
    }
    __device__ __forceinline__ bool all_good(const Paged& c, const Unit& x, int k0) const {
        const int lane = threadIdx.x & 31, last = ((k0 + x.n - 1) >> c.shift) - (k0 >> c.shift);
        return !__any_sync(0xffffffffu, (lane <= last && !c.is_page(a)) || (lane + 32 <= last && !c.is_page(b)));
    }
};

__device__ __forceinline__ ChunkPages load_pages(const Paged& c, const Unit& x, int k0) {
    const int lane = threadIdx.x & 31, last = ((k0 + x.n - 1) >> c.shift) - (k0 >> c.shift);
    const int32_t* row = c.table + static_cast<size_t>(x.b) * c.max_pages + (k0 >> c.shift) + lane;
    ChunkPages g{-1, -1};
    if (lane <= last) g.a = row[0];
    if (lane + 32 <= last) g.b = row[32];
    return g;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, Cut<D>::kCtas)
    attn_units(const Paged c, const AttnParams p, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map) {
    using C = Cut<D>;
    constexpr int kB = D / 16;                  // 16-wide blocks of a row
    constexpr int kMine = D / 64;               // of them a warp's share of the output
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_units[kSegments], s_cost[kSegments], s_sum[kWarps + 1], s_cost_sum[kWarps + 1];
    __shared__ uint4 s_p[kWarps][NT][32];       // probabilities of 16 slots, as operand fragments
    __shared__ float s_top[kWarps][8 * NT], s_l[kWarps][8 * NT];
    __shared__ uint64_t s_full[C::kStages], s_empty[C::kStages];
    __shared__ int s_good[C::kStages];          // the round's unit has no page id out of range
    uint8_t* const smem = smem_raw + (-fer::dev::smem_addr(smem_raw) & 1023u);
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    if (t < C::kStages) {
        fer::dev::mbar_init(&s_full[t], 1);
        fer::dev::mbar_init(&s_empty[t], kWarps);
        fer::dev::fence_mbar_init();
    }
    if (t == 0) {
        fer::dev::prefetch_tmap(&k_map);
        fer::dev::prefetch_tmap(&v_map);
    }
    // lengths and page ids into L2 while the kernel before still runs: only a hint, their values are read behind it
    {
        const size_t line = static_cast<size_t>(blockIdx.x) * kThreads + t, ids = static_cast<size_t>(p.n_seq) * c.max_pages;
        if (line * 32 < ids) fer::dev::prefetch_l2(c.table + line * 32);
        if (line * 32 < static_cast<size_t>(p.n_seq)) fer::dev::prefetch_l2(c.lengths + line * 32);
    }
    fer::dev::pdl_begin();

    // sequences that hold nothing have no unit: their results are written here
    for (int b = blockIdx.x; b < p.n_seq; b += gridDim.x) {
        bool bad;
        const int len = c.length(b, &bad);
        if (bad && t == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
        if (len > 0) continue;
        T* o = static_cast<T*>(p.out) + b * p.os;
        for (int i = t; i < p.heads * D; i += kThreads) o[i] = static_cast<T>(0.0f);
        if (p.lse)
            for (int i = t; i < p.heads; i += kThreads) p.lse[static_cast<size_t>(b) * p.heads + i] = -INFINITY;
    }
    Units table{s_units, s_cost, 0, 0};
    UnitRun run;
    int u0 = 0, u1 = 1;
    if (p.direct) {
        // no table: this CTA's unit by its index
        const int heads = c.kv_heads * p.blocks, chunk = blockIdx.x % p.chunks, hb = blockIdx.x / p.chunks;
        const int b = hb / heads, h = hb - b * heads;
        const Seq q(c, p, b);
        if (chunk >= q.chunks) return;
        run.from = 0;
        run.x = Unit{b, h / p.blocks, h % p.blocks, chunk, q.chunks, min(p.chunk(), q.len - (chunk << p.chunk_log2))};
        __syncthreads();   // the barriers are set up
    } else {
        // how many units each segment of sequences has and what they cost, and the sums before them
        table.seg = (p.n_seq + kSegments - 1) / kSegments;
        table.segments = (p.n_seq + table.seg - 1) / table.seg;
        int cost_carry = 0;
        int carry = 0;
        for (int s0 = 0; s0 < table.segments; s0 += kThreads) {
            int mine = 0;
            int cost = 0;
            const int s = s0 + t;
            if (s < table.segments) {
                for (int b = s * table.seg; b < min(p.n_seq, (s + 1) * table.seg); ++b) {
                    const Seq q(c, p, b);
                    mine += q.units();
                    cost += q.cost();
                }
            }
            int x = mine;
            int y = cost;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int x1 = __shfl_up_sync(0xffffffffu, x, off);
                const int y1 = __shfl_up_sync(0xffffffffu, y, off);
                if (lane >= off) x += x1, y += y1;
            }
            if (lane == 31) s_sum[w] = x, s_cost_sum[w] = y;
            __syncthreads();
            x += carry - mine;
            y += cost_carry - cost;
            for (int i = 0; i <= kWarps; ++i) {
                if (i < w) x += s_sum[i], y += s_cost_sum[i];
                carry += s_sum[i];
                cost_carry += s_cost_sum[i];
            }
            if (s < table.segments) s_units[s] = x, s_cost[s] = y;
            __syncthreads();
        }
        // this CTA's run: the units that begin in its equal part of the whole cost
        {
            const int x = static_cast<int>(static_cast<unsigned long long>(static_cast<unsigned>(cost_carry)) *
                                           (blockIdx.x + (lane & 1)) / gridDim.x);
            const int u = x >= cost_carry ? carry : unit_at(c, p, table, x);
            u0 = __shfl_sync(0xffffffffu, u, 0);
            u1 = __shfl_sync(0xffffffffu, u, 1);
        }
        if (u0 >= u1) return;
    }

    const uint32_t ring = fer::dev::smem_addr(smem);
    bool alive = true;   // no wait of this warp has run out
    if (w == kWarps) {
        // The loading warp: every unit's rounds in order, round q of the run
        // into stage q % kStages. A box is rows of one page, 64 dims, a lane each.
        const int box_rows = min(kRound, c.page_size()), row_boxes = kRound / box_rows;
        const int boxes = 2 * (D / 64) * row_boxes;
        const uint32_t full0 = fer::dev::smem_addr(&s_full[0]);
        // rows that are read once leave L2 first, so the parts and scores stay for the joining
        // (two of 40003 slots with weights 38.3 -> 36.7 us, 131071 slots 95.2 -> 93.3)
        uint64_t policy;
        if (p.blocks == 1) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
        Unit x = run.get(c, p, table, u0, u1 - 1), next = x;
        ChunkPages pages = load_pages(c, x, x.chunk << p.chunk_log2), ahead = pages;
        int q = 0;
        for (int u = u0; u < u1 && alive; ++u) {
            if (u + 1 < u1) {   // the next unit's page ids are on their way meanwhile
                next = run.get(c, p, table, u + 1, u1 - 1);
                ahead = load_pages(c, next, next.chunk << p.chunk_log2);
            }
            const int k0 = x.chunk << p.chunk_log2;
            const int good = pages.all_good(c, x, k0);
            if (!good && lane == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
            for (int r0 = 0; r0 < x.n; r0 += kRound, ++q) {
                const int stage = q % C::kStages;
                alive = __all_sync(0xffffffffu, fer::dev::mbar_wait(&s_empty[stage], (q / C::kStages & 1) ^ 1));
                if (!alive) break;
                if (lane == 0) {
                    s_good[stage] = good;
                    fer::dev::mbar_arrive_expect_tx(&s_full[stage], C::kStage);
                }
                for (int i = lane; i - lane < boxes; i += 32) {
                    const int value = i >= boxes / 2, j = i - value * (boxes / 2);
                    const int band = j % (D / 64), rows = j / (D / 64) * box_rows;
                    // slots of no page are read as page `pages`, which is outside the map: zeros
                    const int slot = r0 + min(rows, kRound - box_rows);
                    const int id = pages.of(c, k0, slot);
                    if (i < boxes)
                        load_box(ring + stage * C::kStage + value * C::kHalf + band * C::kBand + rows * 128,
                                 value ? &v_map : &k_map, band * 64, (k0 + slot) & (c.page_size() - 1), x.hk,
                                 c.is_page(id) ? id : c.pages, full0 + 8 * stage, policy);
                }
            }
            x = next;
            pages = ahead;
        }
        // the copies have landed before this warp leaves, whatever became of the others
        for (int k = max(0, q - C::kStages); k < q; ++k)
            alive = fer::dev::mbar_wait(&s_full[k % C::kStages], k / C::kStages & 1) && alive;
        if (!alive && lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutLoad);
        return;
    }

    // Queries as columns (heads lane / 4) of rows (dims 2 (lane % 4) + {0, 1}
    // and 8 more); columns behind the group's last head repeat its first and are
    // left out at the end. Those of the next unit are loaded a unit ahead
    // where the registers allow it.
    constexpr bool kAhead = NT * kB <= 16;
    uint32_t qf[NT][kB][2], qn[NT][kB][2];
    auto load_q = [&](const Unit& x, uint32_t (&q)[NT][kB][2]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int g = x.blk * 8 * NT + nt * 8 + lane / 4;
            const T* row = static_cast<const T*>(p.q) + x.b * p.qs +
                           (static_cast<size_t>(x.hk) * p.group + (g < p.group ? g : 0)) * D;
            const bool even = (reinterpret_cast<uintptr_t>(row) & 3) == 0;
#pragma unroll
            for (int k = 0; k < kB; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint16_t* at = reinterpret_cast<const uint16_t*>(row + 16 * k + 8 * e + 2 * (lane & 3));
                    uint32_t v;
                    if (even) v = *reinterpret_cast<const uint32_t*>(at);
                    else v = at[0] | static_cast<uint32_t>(at[1]) << 16;
                    q[nt][k][e] = v;
                }
        }
    };
    Unit x = run.get(c, p, table, u0, u1 - 1);
    load_q(x, qf);
    int q = 0;   // rounds of the run so far
    for (int u = u0; u < u1; ++u) {
        const int h0 = x.hk * p.group + x.blk * 8 * NT;          // first head of the block
        const int nh = min(8 * NT, p.group - x.blk * 8 * NT);    // its heads
        const int k0 = x.chunk << p.chunk_log2;
        const Unit next = u + 1 < u1 ? run.get(c, p, table, u + 1, u1 - 1) : x;
        const bool turn = next.b != x.b || next.hk != x.hk || next.blk != x.blk;
        if (kAhead && turn) load_q(next, qn);

        // this lane's heads: 8 nt + 2 (lane % 4) + e. m is the same in all warps, l of this lane's slots
        float m[NT][2], l[NT][2], o[NT][kMine][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int k = 0; k < kMine; ++k) o[nt][k][0] = o[nt][k][1] = o[nt][k][2] = o[nt][k][3] = 0.0f;
        }
        for (int r0 = 0; r0 < x.n; r0 += kRound, ++q) {
            const int stage = q % C::kStages;
            if (alive) alive = fer::dev::mbar_wait(&s_full[stage], q / C::kStages & 1);
            const bool good = s_good[stage];
            const uint32_t st = ring + stage * C::kStage;
            const int rows = x.n - r0;           // held slots of the round, or more
            float s[NT][4];
            {
                float s2[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.0f;
                const int r = 16 * w + (lane & 15);
#pragma unroll
                for (int k = 0; k < kB; ++k) {
                    uint32_t a[4];
                    ldsm4(a, st + C::at(r, 2 * k + (lane >> 4)));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma<T>(k & 1 ? s2[nt] : s[nt], a, qf[nt][k][0], qf[nt][k][1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = (s[nt][e] + s2[nt][e]) * p.scale2;
            }
            const int j = r0 + 16 * w + lane / 4;   // this lane's slots of the chunk: j, j + 8
            bool on0 = j < x.n, on1 = j + 8 < x.n;
            if (!good) {
                const ChunkPages pg = load_pages(c, x, k0);
                const int p0 = pg.of(c, k0, min(j, x.n - 1)), p1 = pg.of(c, k0, min(j + 8, x.n - 1));
                on0 = on0 && c.is_page(p0);
                on1 = on1 && c.is_page(p1);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (!on0) s[nt][e] = -INFINITY;
                    if (!on1) s[nt][2 + e] = -INFINITY;
                    float v = fmaxf(s[nt][e], s[nt][2 + e]);
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                    if (lane < 4) s_top[w][nt * 8 + 2 * lane + e] = v;
                }
            if (p.scores) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int g = nt * 8 + 2 * (lane & 3) + e;
                        float* row = p.scores + (static_cast<size_t>(x.b) * p.heads + h0 + g) * c.max_slots() + k0;
                        if (g < nh && j < x.n) row[j] = s[nt][e];
                        if (g < nh && j + 8 < x.n) row[j + 8] = s[nt][2 + e];
                    }
            }
            meet_warps();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = m[nt][e];
#pragma unroll
                    for (int v = 0; v < kWarps; ++v) top = fmaxf(top, s_top[v][nt * 8 + 2 * (lane & 3) + e]);
                    const float base = top == -INFINITY ? 0.0f : top;
                    const float f = ex2(m[nt][e] - base);   // 1 where the maximum stays
                    m[nt][e] = top;
                    s[nt][e] = ex2(s[nt][e] - base);
                    s[nt][2 + e] = ex2(s[nt][2 + e] - base);
                    l[nt][e] = l[nt][e] * f + (s[nt][e] + s[nt][2 + e]);
#pragma unroll
                    for (int k = 0; k < kMine; ++k) o[nt][k][e] *= f, o[nt][k][2 + e] *= f;
                }
                uint4 f;
                split2<T>(s[nt][0], s[nt][1], f.x, f.z);
                split2<T>(s[nt][2], s[nt][3], f.y, f.w);
                f.x = transpose8(f.x), f.y = transpose8(f.y), f.z = transpose8(f.z), f.w = transpose8(f.w);
                s_p[w][nt][lane] = f;
            }
            meet_warps();
            // the low parts' products in a sum of their own: chains of dependent products half as long
            constexpr bool kTwo = NT == 1;
            float low[NT][kMine][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < kMine; ++k) low[nt][k][0] = low[nt][k][1] = low[nt][k][2] = low[nt][k][3] = 0.0f;
#pragma unroll
            for (int v = 0; v < kWarps; ++v) {
                if (16 * v >= rows) break;
                uint4 f[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) f[nt] = s_p[v][nt][lane];
                const int r = 16 * v + (lane & 7) + ((lane >> 4) << 3);
                const int left = rows - 16 * v - 2 * (lane & 3);   // a lane has slots 0, 1, 8 and 9 from there
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    uint32_t a[4];
                    ldsm4_t(a, st + C::kHalf + C::at(r, 2 * (w * kMine + k) + ((lane >> 3) & 1)));
                    if (16 * v + 16 > rows) {   // values behind the last slot count as zero, whatever is there
                        const uint32_t m0 = left > 1 ? ~0u : left > 0 ? 0xffffu : 0u;
                        const uint32_t m1 = left > 9 ? ~0u : left > 8 ? 0xffffu : 0u;
                        a[0] &= m0, a[1] &= m0, a[2] &= m1, a[3] &= m1;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma<T>(kTwo ? low[nt][k] : o[nt][k], a, f[nt].z, f[nt].w);
                        mma<T>(o[nt][k], a, f[nt].x, f[nt].y);
                    }
                }
            }
            if constexpr (kTwo) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < kMine; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[nt][k][e] += low[nt][k][e];
            }
            __syncwarp();
            if (lane == 0) fer::dev::mbar_arrive(&s_empty[stage]);
        }

        // the unit's sums, and each warp's dims of its result
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
                l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
                if (lane < 4) s_l[w][nt * 8 + 2 * lane + e] = l[nt][e];
            }
        meet_warps();
        const bool whole = x.chunks == 1;
        constexpr float kBack = 1.0f / kScaleP<T>;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int g = nt * 8 + 2 * (lane & 3) + e;
                if (g >= nh) continue;
                float sum = 0.0f;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) sum += s_l[v][g];
                const size_t bh = static_cast<size_t>(x.b) * p.heads + h0 + g, at = bh * p.chunks + x.chunk;
                if (w == 0 && lane < 4) {
                    *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m[nt][e], sum);
                    if (whole && p.lse) p.lse[bh] = sum == 0.0f ? -INFINITY : (m[nt][e] + log2f(sum)) * kLn2;
                }
                const float f = !whole ? kBack : sum == 0.0f ? 0.0f : kBack / sum;
                T* const out = static_cast<T*>(p.out) + x.b * p.os + static_cast<size_t>(h0 + g) * D;
                float* const part = p.part_o + at * D;
#pragma unroll
                for (int k = 0; k < kMine; ++k)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int d = 16 * (w * kMine + k) + 8 * r + lane / 4;
                        const float v = o[nt][k][2 * r + e] * f;
                        if (whole) out[d] = static_cast<T>(sum == 0.0f ? 0.0f : v);
                        else part[d] = v;
                    }
            }
        if (turn) {
            if constexpr (kAhead) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < kB; ++k) qf[nt][k][0] = qn[nt][k][0], qf[nt][k][1] = qn[nt][k][1];
            } else {
                load_q(next, qf);
            }
        }
        x = next;
    }
    if (!alive && lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutLoad);
}

// log2 of a head's total sum of powers, from its chunks' (m, l), by one warp;
// -inf where nothing counts. BATCH loads a lane are in flight.
template <int BATCH>
__device__ __forceinline__ float chunks_lse2(const float* ml, int chunks) {
    const int lane = threadIdx.x & 31;
    float top = -INFINITY, l = 0.0f;
    for (int i0 = lane; i0 < chunks; i0 += 32 * BATCH) {
        float2 v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            v[k] = make_float2(-INFINITY, 0.0f);
            if (i0 + 32 * k < chunks) v[k] = *reinterpret_cast<const float2*>(ml + 2 * (i0 + 32 * k));
        }
        float next = top;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) next = fmaxf(next, v[k].x);
        const float b = next == -INFINITY ? 0.0f : next;
        l *= ex2(top - b);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) l += v[k].y * ex2(v[k].x - b);
        top = next;
    }
    float all = top;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, off));
    const float base = all == -INFINITY ? 0.0f : all;
    l *= ex2(top - base);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    return l == 0.0f ? -INFINITY : base + log2f(l);
}

// grid (group * D / DIMS + weight tiles, kv_heads, n_seq). The first CTAs of a
// (key head, sequence) add one head's chunks for DIMS dims each: a warp takes
// every kW-th chunk in order, DIMS / 32 dims a lane (and again for the next
// start, where the CTA has fewer warps), and these kW sums, each of a maximum
// of its own, are added in order. The others add
// probabilities to the weights of four slots a thread, with what does not
// depend on the total in flight before they wait for it.
template <typename T, int D, int kFinish, int DIMS, int kW>
__global__ void __launch_bounds__(kFinish) attn_finish(const Paged c, const AttnParams p) {
    constexpr int kWarpsIn = kFinish / 32, kV = DIMS / 32, kBands = D / DIMS, kHeads = 4;
    // Chunks that share a maximum, and batches of lse's loads: functions of D and kW, so not of the batch.
    constexpr int kStep = D <= 128 ? 4 : 2, kBatch = kW > 8 ? 8 : 1;
    constexpr int kAhead = kV == 1 ? 16 : kStep;   // chunks in flight
    __shared__ __align__(16) float s_o[kW][DIMS];
    __shared__ float2 s_ml[kW];
    __shared__ float s_lse[kFinish];
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    const int b = blockIdx.z, hk = blockIdx.y;
    fer::dev::pdl_begin();
    bool bad;
    const int len = c.length(b, &bad);
    const int chunks = p.chunks_of(len);
    const size_t bh0 = static_cast<size_t>(b) * p.heads + static_cast<size_t>(hk) * p.group;
    if (static_cast<int>(blockIdx.x) < p.group * kBands) {
        if (chunks <= 1) return;                      // written already
        const int g = blockIdx.x / kBands, d0 = blockIdx.x % kBands * DIMS;
        const size_t bh = bh0 + g;
        const float2* const ml = reinterpret_cast<const float2*>(p.part_ml) + bh * p.chunks;
        struct alignas(4 * (kV < 4 ? kV : 4)) Dims { float e[kV]; };
        const float* const po = p.part_o + bh * p.chunks * D + d0 + kV * lane;
        for (int part = w; part < kW; part += kWarpsIn) {
            float top = -INFINITY, l = 0.0f;
            Dims o{};
            for (int i0 = part; i0 < chunks; i0 += kW * kAhead) {
                Dims v[kAhead];
                float2 x[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int i = i0 + k * kW;
                    x[k] = make_float2(-INFINITY, 0.0f);
                    v[k] = Dims{};
                    if (i < chunks) x[k] = ml[i], v[k] = *reinterpret_cast<const Dims*>(po + static_cast<size_t>(i) * D);
                }
#pragma unroll
                for (int k0 = 0; k0 < kAhead; k0 += kStep) {
                    float next = top;
#pragma unroll
                    for (int k = k0; k < k0 + kStep; ++k) next = fmaxf(next, x[k].x);
                    const float base = next == -INFINITY ? 0.0f : next, f = ex2(top - base);
                    l *= f;
#pragma unroll
                    for (int e = 0; e < kV; ++e) o.e[e] *= f;
#pragma unroll
                    for (int k = k0; k < k0 + kStep; ++k) {
                        const float y = ex2(x[k].x - base);
                        l = fmaf(x[k].y, y, l);
#pragma unroll
                        for (int e = 0; e < kV; ++e) o.e[e] = fmaf(v[k].e[e], y, o.e[e]);
                    }
                    top = next;
                }
            }
            *reinterpret_cast<Dims*>(&s_o[part][kV * lane]) = o;
            if (lane == 0) s_ml[part] = make_float2(top, l);
        }
        __syncthreads();
        if (t >= DIMS) return;
        float all = -INFINITY, sum = 0.0f, out = 0.0f;
#pragma unroll
        for (int i = 0; i < kW; ++i) all = fmaxf(all, s_ml[i].x);
        const float base = all == -INFINITY ? 0.0f : all;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            const float y = ex2(s_ml[i].x - base);
            sum = fmaf(s_ml[i].y, y, sum);
            out = fmaf(s_o[i][t], y, out);
        }
        static_cast<T*>(p.out)[b * p.os + (static_cast<size_t>(hk) * p.group + g) * D + d0 + t] =
            static_cast<T>(sum == 0.0f ? 0.0f : out / sum);
        if (d0 + t == 0 && p.lse) p.lse[bh] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * kLn2;
        return;
    }
    const size_t most = static_cast<size_t>(c.max_slots());   // a multiple of 8: rows start at 16 bytes
    const uint32_t step = (gridDim.x - p.group * kBands) * 4 * kFinish;   // j0 may pass 31 bits at the end
    for (uint32_t j0 = (blockIdx.x - p.group * kBands) * 4 * kFinish; j0 < static_cast<uint32_t>(len); j0 += step) {
        const int j = static_cast<int>(j0) + 4 * t;
        const bool on = j < len, whole = j + 3 < len && reinterpret_cast<uintptr_t>(p.weights) % 16 == 0;
        const float* const scores = p.scores + bh0 * most + j;
        float* const out = p.weights + (static_cast<size_t>(b) * c.kv_heads + hk) * most + j;
        float4 s[kHeads], old = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (whole) old = *reinterpret_cast<const float4*>(out);
#pragma unroll
        for (int k = 0; k < kHeads; ++k)
            if (on && k < p.group) s[k] = *reinterpret_cast<const float4*>(scores + k * most);
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int g0 = 0; g0 < p.group; g0 += kFinish) {
            const int ng = min(kFinish, p.group - g0);
            if (p.group > kFinish || j0 < step) {   // else the totals are there from the first tile
                __syncthreads();
                for (int g = w; g < ng; g += kWarpsIn) {
                    const float v = chunks_lse2<kBatch>(p.part_ml + 2 * (bh0 + g0 + g) * p.chunks, chunks);
                    if (lane == 0) s_lse[g] = v;
                }
                __syncthreads();
            }
            if (!on) continue;
            for (int g = 0; g < ng; g += kHeads) {
#pragma unroll
                for (int k = 0; k < kHeads; ++k)
                    if ((g0 > 0 || g > 0) && g + k < ng)
                        s[k] = *reinterpret_cast<const float4*>(scores + (g0 + g + k) * most);
#pragma unroll
                for (int k = 0; k < kHeads; ++k) {
                    if (g + k >= ng) break;
                    const float lse2 = s_lse[g + k];
                    if (lse2 == -INFINITY) continue;
                    sum[0] += ex2(s[k].x - lse2);
                    sum[1] += ex2(s[k].y - lse2);
                    sum[2] += ex2(s[k].z - lse2);
                    sum[3] += ex2(s[k].w - lse2);
                }
            }
        }
        if (whole) {
            *reinterpret_cast<float4*>(out) = make_float4(old.x + sum[0], old.y + sum[1], old.z + sum[2], old.w + sum[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < len) out[e] += sum[e];
        }
    }
}

// CTAs of a kernel that fit on the current device at once; 0 on an error. The
// answer is kept per device, where the shared-memory limit is also set.
int resident(const void* kernel, int smem, std::atomic<int>* known) {
    int dev = 0, n = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= fer::host::kMaxDevices) return 0;
    if (const int k = known[dev].load(std::memory_order_relaxed)) return k;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, smem) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    known[dev].store(n * sms, std::memory_order_relaxed);
    return n * sms;
}

// Boxes of 64 dims x `rows` rows of one page; 128-byte swizzle.
bool map_pages(CUtensorMap* m, const Paged& c, void* base, uint32_t dtype, int rows) {
    const fer::host::EncodeTiledFn fn = fer::host::encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t page = static_cast<cuuint64_t>(c.page_size()), row = 2ull * c.head_dim;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), page, static_cast<cuuint64_t>(c.kv_heads),
                                static_cast<cuuint64_t>(c.pages)};
    const cuuint64_t strides[3] = {row, page * row, page * row * c.kv_heads};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, step[4] = {1, 1, 1, 1};
    return fn(m, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides,
              box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int THREADS, int DIMS, int kW>
cudaError_t finish(const Paged& c, const AttnParams& p, cudaStream_t s) {
    // as many tiles a (key head, sequence) as there are, within kTiles CTAs: a wide table has mostly empty ones
    // (those 64 x 32 heads with weights: 66 us in all with every tile its CTA, 37 so)
    const long long pairs = static_cast<long long>(c.kv_heads) * p.n_seq;
    const int all = p.weights ? (c.max_slots() - 1) / (4 * THREADS) + 1 : 0, least = static_cast<int>(kTiles / pairs) + 1;
    const int tiles = all < least ? all : least;
    return fer::host::launch_pdl(attn_finish<T, D, THREADS, DIMS, kW>,
                                 dim3(p.group * (D / DIMS) + tiles, c.kv_heads, p.n_seq), dim3(THREADS), 0, s, c, p);
}

template <typename T, int D, int NT>
cudaError_t run(const Paged& c, AttnParams& p, cudaStream_t s) {
    constexpr int smem = Cut<D>::kSmem;
    static std::atomic<int> known[fer::host::kMaxDevices];
    const int ctas = resident(reinterpret_cast<const void*>(attn_units<T, D, NT>), smem, known);
    if (ctas <= 0) return cudaErrorInvalidConfiguration;
    CUtensorMap k_map, v_map;
    const int rows = kRound < c.page_size() ? kRound : c.page_size();
    const uint32_t dtype = __is_same(T, __half) ? 1 : 2;
    if (!map_pages(&k_map, c, c.k, dtype, rows) || !map_pages(&v_map, c, c.v, dtype, rows)) return cudaErrorInvalidValue;
    const long long most = static_cast<long long>(p.n_seq) * c.kv_heads * p.blocks * p.chunks;
    p.direct = most <= ctas;
    cudaError_t e = fer::host::launch_pdl(attn_units<T, D, NT>, dim3(static_cast<unsigned>(most < ctas ? most : ctas)),
                                          dim3(kThreads), smem, s, c, p, k_map, v_map);
    if (e == cudaSuccess && (p.weights || p.chunks > 1)) {
        // few chunks or many heads: a head a CTA; else sixteen warps for 32 dims, whose loads one SM could not have
        // in flight (256 chunks: 8.9 us with a head a CTA, 6.0 so; 4 chunks: 6.2 so, 5.2 with a head a CTA; 64 x 32
        // heads of up to 512 slots in a table of 32768: 52 us in all so, 33 with a head a CTA)
        // Which warp takes which chunk, and with it every rounding, is a function of the table's width.
        if (p.chunks <= 32) e = finish<T, D, 256, D, 8>(c, p, s);
        else if (static_cast<long long>(p.n_seq) * p.heads >= kManyHeads) e = finish<T, D, 256, D, 16>(c, p, s);
        else e = finish<T, D, 512, 32, 16>(c, p, s);
    }
    return e;
}

// Head blocks a key head: of up to 8 heads, or of up to 16 where it has more.
int blocks_of(int group) { return group <= 8 ? 1 : (group - 1) / 16 + 1; }

template <typename T, int D>
cudaError_t run_heads(const Paged& c, AttnParams& p, cudaStream_t s) {
    return p.group <= 8 ? run<T, D, 1>(c, p, s) : run<T, D, 2>(c, p, s);
}

template <typename T>
cudaError_t run_dim(const Paged& c, AttnParams& p, cudaStream_t s) {
    switch (c.head_dim) {
        case 64: return run_heads<T, 64>(c, p, s);
        case 128: return run_heads<T, 128>(c, p, s);
        default: return run_heads<T, 256>(c, p, s);
    }
}

size_t up16(size_t v) { return (v + 15) & ~size_t(15); }

}  // namespace

extern "C" size_t fer_paged_attention_workspace_bytes(int n_seq, int heads, int kv_heads, int head_dim, int max_slots,
                                                      int with_weights) {
    if (n_seq <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_slots <= 0) return 0;
    const size_t bh = static_cast<size_t>(n_seq) * heads;
    const size_t chunks = (max_slots - 1) / chunk_of(max_slots) + 1;
    size_t n = up16(bh * chunks * 2 * sizeof(float)) + up16(bh * chunks * head_dim * sizeof(float));
    if (with_weights) n += up16(bh * max_slots * sizeof(float));
    return n;
}

extern "C" cudaError_t fer_paged_attention(const fer_paged_view_t* cache, const fer_paged_attention_args_t* a,
                                           uint32_t* err, cudaStream_t s) {
    Paged c{};
    const cudaError_t ce = fer::host::paged_params(cache, &c);
    if (ce != cudaSuccess) return ce;
    if (!a || !a->q || !a->out || a->n_seq < 0 || a->n_seq > cache->batch || a->heads <= 0 || a->heads % c.kv_heads)
        return cudaErrorInvalidValue;
    const size_t width = static_cast<size_t>(a->heads) * c.head_dim;
    if (a->q_stride < width || a->out_stride < width || !(a->scale >= 0.0f) || a->scale > kMostScale)
        return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % 2) return cudaErrorInvalidValue;
    if (!fer::host::words_aligned({a->lse, a->weights})) return cudaErrorInvalidValue;
    if (a->n_seq == 0) return cudaSuccess;
    if (c.kv_heads > 65535 || a->n_seq > 65535) return cudaErrorNotSupported;
    const int max_slots = c.max_slots();
    // units and their cost are counted in 31 bits
    const int group = a->heads / c.kv_heads;
    const long long blocks = static_cast<long long>(a->n_seq) * c.kv_heads * blocks_of(group);
    if (blocks * (rounds_of(max_slots) + kUnitCost * ((max_slots - 1ll) / chunk_of(max_slots) + 1)) > 0x7fffffffll)
        return cudaErrorNotSupported;
    const size_t need = fer_paged_attention_workspace_bytes(a->n_seq, a->heads, c.kv_heads, c.head_dim, max_slots,
                                                            a->weights != nullptr);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need)
        return cudaErrorInvalidValue;
    AttnParams p{};
    p.q = a->q;
    p.out = a->out;
    p.qs = a->q_stride;
    p.os = a->out_stride;
    p.n_seq = a->n_seq;
    p.heads = a->heads;
    p.group = group;
    p.blocks = blocks_of(group);
    while ((1 << p.chunk_log2) < chunk_of(max_slots)) ++p.chunk_log2;
    p.chunks = (max_slots - 1) / chunk_of(max_slots) + 1;
    p.scale2 = (a->scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(c.head_dim)) : a->scale) * kLog2e;
    p.lse = a->lse;
    p.weights = a->weights;
    p.err = err;
    const size_t bh = static_cast<size_t>(a->n_seq) * a->heads;
    char* w = static_cast<char*>(a->workspace);
    p.part_ml = reinterpret_cast<float*>(w);
    w += up16(bh * p.chunks * 2 * sizeof(float));
    p.part_o = reinterpret_cast<float*>(w);
    w += up16(bh * p.chunks * c.head_dim * sizeof(float));
    if (a->weights) p.scores = reinterpret_cast<float*>(w);
    return cache->dtype == 1 ? run_dim<__half>(c, p, s) : run_dim<__nv_bfloat16>(c, p, s);
}
