// Attention over a paged key-value cache in tensor-core tiles: rows of prompts or
// single tokens with a sliding window and sinks, and a batch of single tokens
// behind a prefix that all of them share.
//
// A row is one query head of one token. The rows that read the same keys, those
// of one key head, lie side by side: token by token, each with its group of
// query heads. A unit of work is up to 256 rows (two sub-tiles of 128, the
// lanes of tensor memory; one of 128 where head_dim is 256) and a range of key
// blocks. Per block S = Q K^T, P = 2^(scale S - m) and O += P V; a row's m, l = sum
// P and O stay on chip for the whole range: 4 flops a row, slot and dim, and
// each key and value is read once a unit. 256 rows a unit are 256 flops a byte
// of keys and values, which is what the GPU's tensor rate needs of its HBM rate.
//
// Warps. One finds units, one ahead of the others, and loads their queries; one
// loads keys and values by tensor copies of page rows into a ring of tiles,
// running on into the next unit; one for each sub-tile issues its products: P V
// of 64 keys, then S of the 64 after next, so that S of the next 64 is there
// while P of these is computed. Four warps take a sub-tile's softmax, a row a
// thread, 64 keys at a time. P replaces S in tensor memory and is the left
// operand from there. The maximum a row subtracts is raised only when a block's
// exceeds it by 2^kSlack (softmax does not depend on it), so O is seldom
// rescaled. Where a unit has more than 128 rows each sub-tile has its own, and
// their exponentials take turns. Where it has at most 128 the two sub-tiles are
// the same rows with every other key block each, added up at the end: single
// tokens keep both in flight; and of at most kFew rows each is in all four
// quarters of a sub-tile, which share the keys' exponentials and P's bits.
//
// What bounds it. Wide units: the latency of a sub-tile's 64 keys (scores from
// tensor memory, maximum, exponentials, P back, about 1900 cycles, while the
// tensor cores are busy 58% of the time and the issue slots 45%): a piece of 4001
// tokens behind 28000, 32 heads x 128, takes 1940 to 1998 us, 984 to 1013 TFLOP/s.
// Loops that stay in the instruction cache matter as much as their length
// (prompts behind a window 478 -> 372 us by chunks that are looped over instead
// of unrolled). Prompts behind a window of 512 (320 to 345 us for 16 of up to
// 2048) lose a third to masked blocks, whose slots are tested one by one, and
// 6000 cycles a unit to its results. Units of few rows: latency and uneven
// shares (3.2 TB/s); where all rows are single tokens of small groups, and
// where own slots behind a prefix are many, the kernel of one-token attention
// takes them, which has three or four small CTAs an SM.
//
// P is rounded to 16 bits once, by half a step of the type at most, and l sums it
// unrounded; where rows are few (kFine) what rounding leaves is multiplied as a
// second operand, as the tensor cores wait for memory there anyway. P of f16 is
// held 2^kUp higher, so that what rounds to 0 is below 2^-33 of the largest.
//
// Units are numbered from the lengths on the device, and CTA i of G takes i, 2G -
// 1 - i, 2G + i, ...: sequences in their order, and of a sequence's key head the
// longest first (32 causal prompts of 128 to 4096 tokens, 32 / 8 heads x 128:
// 1706 us with the longest prompt last, 1781 with it first). Which CTA takes a unit
// does not change its arithmetic. Where rows are few for the GPU a row's keys
// are cut into several units, whose m, l and O go to the workspace in f32, and
// a second kernel adds them in order; cuts are a function of the call's sizes. They
// go by the mean of rows a sequence, so beside a long prompt single tokens may stay
// whole (63 tokens behind 8192 slots 386 us, a prompt of 1024 26, both 395; 127 and
// 4096: 729, 228, both 869 with nothing cut).
//
// Pages without a visible slot are not looked up, and their keys and values are
// zeros. In the value tiles slots that no row of a unit sees become 0, and
// infinities and NaN of slots that some rows see and others do not, for which P =
// 0 would give NaN, are taken out and added to the results of the rows that see
// them. An infinite value whose own probability is 0 in P's type gives NaN, as
// 0 x inf in any softmax of that precision; a score of +inf or NaN makes its row NaN.
#include "f32x2.cuh"
#include "paged.cuh"
#include "pdl.cuh"
#include "tmap.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

namespace {

using fer::dev::Paged;

constexpr int kSms = 148;
constexpr int kSegments = 128;       // entries of the unit table
constexpr int kUnitSlots = 3;        // units handed from the loading warp to the others
constexpr int kBadRing = 16;         // key blocks whose flag is kept
constexpr int kJoinWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMostScale = 2.0e38f;   // times log2 e it is still finite
constexpr float kSlack = 7.0f;          // log2 units the subtracted maximum may lag
// Of so many pairs of exponentials so many go to the multipliers: a long causal piece takes 1985 us with none, 1940 with one of
// 16, 1948 of 8, 1958 of 4 (the sub-tiles' turns hide most of what the unit for exponentials takes).
constexpr int kPoly = 1, kPolyOf = 16;

// Sizes of a head_dim: keys a block, sub-tiles of rows, tiles of the ring.
template <int D> struct Cut {
    static constexpr int kKeys = D == 256 ? 64 : 128;
    static constexpr int kSubs = D == 256 ? 1 : 2;
    static constexpr int kRows = 128 * kSubs;
    static constexpr int kBands = D / 64;
    static constexpr int kTile = kKeys * D * 2;
    static constexpr int kBand = kKeys * 128;        // 64 dims of a tile's keys
    static constexpr int kStages = D == 64 ? 8 : 4;
    static constexpr int kQ = 128 * D * 2;           // queries of a sub-tile
    static constexpr int kSoft = 4 * kSubs;          // softmax warps
    static constexpr int kParts = kKeys / 64;        // 64 keys at a time
    // Softmax warps, one that loads keys and values, one for each sub-tile that issues products, one that loads queries.
    // Registers: of 168 a thread at launch the two groups of four softmax warps take 208 and leave the third group's warps
    // 88. (One group has enough at launch.)
    static constexpr bool kShift = kSubs == 2;
    static constexpr int kThreads = 32 * (kSoft + kSubs + 2);
    static constexpr int kRing = kSubs * kQ;         // where the ring begins
    static constexpr int kMeet = kRing + kStages * kTile;   // 32 KB in which results are added up and turned round
    static constexpr int kSmem = kMeet + 32768 + 1024;
    static constexpr uint32_t kColO = 256;           // O of sub-tile x at kColO + x D, S and P of 64 keys at 128 x and 128 x + 64
    // rows up to which P's rounding is made up for
    static constexpr int kFine = kSubs == 2 ? 128 : 64;
};
constexpr int kUnitBlocks = 3;   // a unit's queries, first scores and results take about as long as so many blocks
constexpr int kFew = 32;   // rows that the four warps of a sub-tile share

// How queries are loaded: 128 (or 32) rows by a tensor copy where the group divides 32, or 128 where no unit has few rows; row
// by row for other groups; by ordinary loads where the addresses are not multiples of 16 bytes.
enum { kQBoxes, kQRows, kQLoads };

// Division of numbers below 2^31 by one divisor, by a product and a shift (Granlund and Montgomery 1994).
struct Divide {
    uint32_t by, mul, shift;
    __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift);
    }
};

struct TileParams {
    const void* q;
    void* out;
    size_t qs, os;
    float* lse;
    const int32_t* offsets;        // null: row b is sequence b's latest slot
    int n_seq, rows, heads, group;
    Divide by_group;
    int window, sinks;             // INT_MAX: no window
    float scale2;                  // scale * log2 e
    int q_maps;                    // kQBoxes, kQRows or kQLoads
    int chunk;                     // key blocks a unit
    int parts;                     // parts a row may have; 0: results go to out
    float* part_ml;                // [rows * heads][parts][2]
    float* part_o;                 // [rows * heads][parts][head_dim]
    int* broken;                   // parts of rows with offsets: whether those cannot be, for the joining
    const int32_t* prefix_pages;   // null: no prefix
    const int32_t* prefix_length;
    int prefix_max, prefix_chunk, own_parts;
    int own_chunk_log2;            // >= 0: sequences' own slots are another kernel's parts, in chunks of 2^that
    const float* own_ml;           // [rows * heads][own_parts][2]
    const float* own_o;
    uint32_t* err;
};

// Some rows of one sequence (or of the whole batch, before the prefix), one key
// head and a range of key blocks.
struct Unit {
    int tok0;          // row of q of the first token; < 0: no more units
    int f0, nf;        // rows: token (f0 + i) / group, head hk * group + (f0 + i) % group
    int hk, seq;       // seq -1: the prefix
    int slot0;         // the first token's slot
    int hi, lo, sink;  // visible to some row: slots below hi that are below sink or not below lo
    int all_hi, all_lo;   // to every row: those below all_hi that are below sink or not below all_lo
    int sb, wb0;       // key blocks: 0 .. sb - 1, then wb0 ..
    int c0, c1;        // of them, counted in that order, the unit's
    int part;          // -1: the only one of its rows
    bool last;         // of the CTA's
};

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

struct Seq {
    int len, n, tok0;
    bool bad, broken;   // its length, its rows out of range
    __device__ __forceinline__ Seq(const Paged& c, const TileParams& p, int b) {
        len = c.length(b, &bad);
        tok0 = b;
        n = 1;
        broken = false;
        if (p.offsets) {
            const int lo = p.offsets[b], hi = p.offsets[b + 1];
            tok0 = min(max(lo, 0), p.rows);
            n = min(max(hi, tok0), p.rows) - tok0;
            broken = tok0 != lo || tok0 + n != hi;
        }
    }
    __device__ __forceinline__ int tiles(const TileParams& p, int rows) const {
        return static_cast<int>((static_cast<long long>(n) * p.group + rows - 1) / rows);
    }
};

// The visible range and the key blocks of tile i of a sequence; returns how many blocks.
template <int D>
__device__ __forceinline__ int tile_range(const TileParams& p, const Seq& q, int i, Unit& u) {
    using C = Cut<D>;
    u.tok0 = q.tok0;
    u.f0 = i * C::kRows;
    u.nf = static_cast<int>(min(static_cast<long long>(C::kRows), static_cast<long long>(q.n) * p.group - u.f0));
    u.slot0 = q.len - q.n;
    const int first = u.slot0 + p.by_group(u.f0), last = u.slot0 + p.by_group(u.f0 + u.nf - 1);
    u.hi = max(last + 1, 0);
    u.all_hi = max(first + 1, 0);
    // rows may lie before slot 0, so that a difference to the window could pass 32 bits
    u.lo = p.window == INT_MAX ? 0 : max(u.all_hi - p.window, 0);
    u.all_lo = p.window == INT_MAX ? 0 : max(u.hi - p.window, 0);
    u.sink = min(p.sinks, u.hi);
    const int end = (u.hi + C::kKeys - 1) / C::kKeys;
    u.wb0 = min(u.lo / C::kKeys, end);
    u.sb = min((u.sink + C::kKeys - 1) / C::kKeys, u.wb0);
    return u.sb + end - u.wb0;
}

__device__ __forceinline__ int chunks_of(int blocks, int chunk) { return blocks <= chunk ? 1 : (blocks - 1) / chunk + 1; }

// Units of one key head of a sequence.
template <int D>
__device__ __forceinline__ int units_of(const TileParams& p, const Seq& q) {
    const int tiles = q.tiles(p, Cut<D>::kRows);
    if (p.parts == 0) return tiles;
    int n = 0;
    for (int i = 0; i < tiles; ++i) {
        Unit u;
        n += chunks_of(tile_range<D>(p, q, i, u), p.chunk);
    }
    return n;
}

// What the prefix is cut into.
template <int D>
struct Prefix {
    int len = 0, tiles = 0, chunks = 0;
    bool bad = false;
    __device__ __forceinline__ Prefix(const Paged& c, const TileParams& p) {
        if (!p.prefix_pages) return;
        const int n = p.prefix_length[0], most = p.prefix_max << c.shift;
        bad = n < 0 || n > most;
        len = min(max(n, 0), most);
        tiles = static_cast<int>((static_cast<long long>(p.n_seq) * p.group + Cut<D>::kRows - 1) / Cut<D>::kRows);
        chunks = len > 0 ? chunks_of((len - 1) / Cut<D>::kKeys + 1, p.prefix_chunk) : 0;
    }
    __device__ __forceinline__ int units(const Paged& c) const { return c.kv_heads * tiles * chunks; }
};

// Whether every sequence has the same number of units, whatever its length: they need not be counted.
__device__ __forceinline__ bool alike(const TileParams& p) { return !p.offsets && p.chunk == INT_MAX; }

// Unit x of the call; s_units: units before every segment of seg sequences, where they are not alike.
template <int D>
__device__ __forceinline__ Unit find_unit(const Paged& c, const TileParams& p, const Prefix<D>& pre, const int* s_units,
                                          int segments, int seg, int x, bool& bad) {
    using C = Cut<D>;
    Unit u{};
    bad = false;
    if (x < pre.units(c)) {
        // tiles that read the same keys next to one another
        const int t = x % pre.tiles, rest = x / pre.tiles, k = rest % pre.chunks;
        u.hk = rest / pre.chunks;
        u.seq = -1;
        u.f0 = t * C::kRows;
        u.nf = static_cast<int>(min(static_cast<long long>(C::kRows), static_cast<long long>(p.n_seq) * p.group - u.f0));
        u.hi = u.all_hi = pre.len;
        const int blocks = (pre.len - 1) / C::kKeys + 1;
        u.c0 = k * p.prefix_chunk;
        u.c1 = min(blocks, u.c0 + p.prefix_chunk);
        u.part = (p.own_chunk_log2 >= 0 ? 0 : p.own_parts) + k;
        return u;
    }
    x -= pre.units(c);
    if (alike(p)) {
        const int tiles = (p.group - 1) / C::kRows + 1, rest = x / tiles;
        u.seq = rest / c.kv_heads;
        u.hk = rest - u.seq * c.kv_heads;
        const Seq q(c, p, u.seq);
        bad = q.bad;
        u.c1 = tile_range<D>(p, q, x - rest * tiles, u);
        u.part = p.prefix_pages ? 0 : -1;
        return u;
    }
    int lo = 0, hi = segments;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_units[mid] <= x) lo = mid;
        else hi = mid;
    }
    x -= s_units[lo];
    int b = lo * seg;
    Seq q(c, p, b);
    int each = units_of<D>(p, q);
    while (x >= each * c.kv_heads && b + 1 < p.n_seq) {
        x -= each * c.kv_heads;
        q = Seq(c, p, ++b);
        each = units_of<D>(p, q);
    }
    u.seq = b;
    u.hk = x / each;
    x -= u.hk * each;
    const int tiles = q.tiles(p, C::kRows);
    int i = tiles - 1;   // the last tile sees most
    int blocks;
    if (p.parts == 0) {
        i -= x;
        blocks = tile_range<D>(p, q, i, u);
        u.c1 = blocks;
        u.part = -1;
        return u;
    }
    for (;; --i) {
        blocks = tile_range<D>(p, q, i, u);
        const int n = chunks_of(blocks, p.chunk);
        if (x < n || i == 0) {
            u.c0 = x * p.chunk;
            u.c1 = min(blocks, u.c0 + p.chunk);
            u.part = n == 1 && !p.prefix_pages ? -1 : x;
            return u;
        }
        x -= n;
    }
}

__device__ __forceinline__ int block_of(const Unit& u, int i) { return i < u.sb ? i : u.wb0 + (i - u.sb); }
// How a unit's blocks are shared: every other one to each sub-tile, or all to both.
template <int D>
__device__ __forceinline__ bool alternate(const Unit& u) { return Cut<D>::kSubs == 2 && u.nf <= 128; }

// Whether the keys of two blocks come before the first's values: K_0 K_1 V_0 K_2 V_1 ... and not K_0 V_0 K_1 V_1 ...
template <int D>
__device__ __forceinline__ bool loads_two(const Unit& u) { return Cut<D>::kSubs == 1 || u.nf <= 128; }
// Place in the ring, from the unit's first, of a block's values.
__device__ __forceinline__ int at_v(bool two, int i, int nb) { return two ? min(2 * i + 2, nb + i) : 2 * i + 1; }

template <int STAGES>
struct Shared {
    uint64_t full[STAGES], empty[STAGES];
    uint64_t unit_full[kUnitSlots], unit_empty[kUnitSlots];
    uint64_t q_full[2], q_empty[2], s_full[2][2], p_full[2][2], o_full[2][2];
    Unit unit[kUnitSlots];
    int bad[kBadRing];
    int units[kSegments], sum[12];
    uint32_t tmem;
    int stop;
    int odd[2];       // infinities or NaN were taken out of the values of an even or odd unit
};

__device__ __forceinline__ void load_q(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(fer::dev::smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int r, int head, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r), "r"(head), "r"(page), "r"(fer::dev::smem_addr(bar))
        : "memory");
}

// 256 threads x 208 and 128 x 88 are the 384 x 168 of the launch.
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }

// Shared-memory matrix descriptors, 128-byte swizzle, 1024 bytes from eight rows to the next: the upper word is the same for
// all, the lower has the address and the bytes from one band to the next, so a step along the tile is one addition.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t at, uint32_t band) { return ((at >> 4) & 0x3FFFu) | ((band >> 4) & 0x3FFFu) << 16; }
// kind::f16, f32 sums, M = 128: N, type of both operands, and whether B has N as its contiguous dimension.
__host__ __device__ constexpr uint32_t idesc(int n, bool bf16, bool b_by_n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_by_n ? 1u << 16 : 0u) | (static_cast<uint32_t>(n) >> 3) << 17 |
           (128u >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tmov.b64 y, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
        : "memory");
}
// One thread of the warp, the same every time.
__device__ __forceinline__ bool elected() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on != 0;
}
// A value that the warp's threads share, known to be one.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(fer::dev::smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this thread's lane of tensor memory; there after wait_ld.
__device__ __forceinline__ void tmem_ld(uint32_t at, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]),
          "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]),
          "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(at)
        : "memory");
}
// The loads into v have landed; v passes through the statements, so that no use comes before them.
template <int N>
__device__ __forceinline__ void wait_ld(float (&v)[N][32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < N; ++j)
        asm volatile(""
                     : "+f"(v[j][0]), "+f"(v[j][1]), "+f"(v[j][2]), "+f"(v[j][3]), "+f"(v[j][4]), "+f"(v[j][5]), "+f"(v[j][6]),
                       "+f"(v[j][7]), "+f"(v[j][8]), "+f"(v[j][9]), "+f"(v[j][10]), "+f"(v[j][11]), "+f"(v[j][12]),
                       "+f"(v[j][13]), "+f"(v[j][14]), "+f"(v[j][15]), "+f"(v[j][16]), "+f"(v[j][17]), "+f"(v[j][18]),
                       "+f"(v[j][19]), "+f"(v[j][20]), "+f"(v[j][21]), "+f"(v[j][22]), "+f"(v[j][23]), "+f"(v[j][24]),
                       "+f"(v[j][25]), "+f"(v[j][26]), "+f"(v[j][27]), "+f"(v[j][28]), "+f"(v[j][29]), "+f"(v[j][30]),
                       "+f"(v[j][31])
                     :
                     : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
// 16 columns; completed by wait_st
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// NaN if one of them is.
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t u;
    if constexpr (__is_same(T, __half)) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
    return u;
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t u, float& lo, float& hi) {
    if constexpr (__is_same(T, __half)) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u));
        lo = v.x, hi = v.y;
    } else {
        lo = __uint_as_float(u << 16), hi = __uint_as_float(u & 0xffff0000u);
    }
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, fer::dev::mbar_wait(bar, parity & 1u));
}
template <int N>
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); }

// The same, and whether some thread says so.
template <int N>
__device__ __forceinline__ bool meet_or(bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"(static_cast<uint32_t>(v)), "n"(N)
                 : "memory");
    return r != 0;
}

// The bits below n, all or none of them where n is past the ends.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// Whether some row of a unit sees a slot of the page.
__device__ __forceinline__ bool page_needed(const Paged& c, const Unit& u, int page) {
    const int first = page << c.shift, last = first + c.page_size() - 1;
    return first < u.hi && (last >= u.lo || first < u.sink);
}
__device__ __forceinline__ const int32_t* table_of(const Paged& c, const TileParams& p, const Unit& u) {
    return u.seq < 0 ? p.prefix_pages : c.table + static_cast<size_t>(u.seq) * c.max_pages;
}
// A row's slots: below end, and below sink or not below begin.
struct Sees {
    int begin, end, sink;
    __device__ __forceinline__ Sees(const TileParams& p, const Unit& u, int f) {
        end = u.seq < 0 ? u.hi : u.slot0 + p.by_group(u.f0 + f) + 1;
        begin = p.window == INT_MAX || u.seq < 0 ? 0 : max(max(end, 0) - p.window, 0);
        sink = p.sinks;
    }
    __device__ __forceinline__ bool operator()(int s) const { return s < end && (s >= begin || s < sink); }
};
__device__ __forceinline__ size_t q_row(const TileParams& p, const Unit& u, int f) {
    return static_cast<size_t>(u.tok0) + p.by_group(u.f0 + f);
}
__device__ __forceinline__ int q_head(const TileParams& p, const Unit& u, int f) {
    return u.hk * p.group + (u.f0 + f) - p.by_group(u.f0 + f) * p.group;
}

// 2^t for two t of at most 126, on the multipliers and adders: t = n + f with |f| <= 1/2, n by rounding in the last bits of
// an f32, 2^f by the polynomial of degree 4 with the least relative error (2.9e-6) among those with 2^0 = 1, and n added to
// its exponent. Below -127 it gives 0.
__device__ __forceinline__ void powers2(uint64_t t2, float& a, float& b) {
    float t0, t1;
    fer::dev::f2_unpack(t2, t0, t1);
    const uint64_t t = fer::dev::f2_pack(fmaxf(t0, -127.0f), fmaxf(t1, -127.0f));
    const uint64_t r = fer::dev::f2_add(t, fer::dev::f2_splat(12582912.0f));
    const uint64_t f = fer::dev::f2_sub(t, fer::dev::f2_sub(r, fer::dev::f2_splat(12582912.0f)));
    uint64_t y = fer::dev::f2_fma(f, fer::dev::f2_splat(0.009582853f), fer::dev::f2_splat(0.055906426f));
    y = fer::dev::f2_fma(y, f, fer::dev::f2_splat(0.24024099f));
    y = fer::dev::f2_fma(y, f, fer::dev::f2_splat(0.69312418f));
    y = fer::dev::f2_fma(y, f, fer::dev::f2_splat(1.0f));
    float r0, r1, y0, y1;
    fer::dev::f2_unpack(r, r0, r1);
    fer::dev::f2_unpack(y, y0, y1);
    a = __uint_as_float(__float_as_uint(y0) + (__float_as_uint(r0) << 23));
    b = __uint_as_float(__float_as_uint(y1) + (__float_as_uint(r1) << 23));
}

template <typename T>
__device__ __forceinline__ void put(T* to, float v) { *to = static_cast<T>(v); }

// Whether some row of the unit does not see a slot that others, or none, see: P is 0 there, and 0 x inf would be NaN.
__device__ __forceinline__ bool hidden(const Unit& u, int s) { return s >= u.all_hi || (s < u.all_lo && s >= u.sink); }
template <int D>
__device__ __forceinline__ bool any_hidden(const Unit& u, int s0, int n) {
    return s0 + n > u.all_hi || (s0 < u.all_lo && s0 + n > u.sink);
}
// The upper bits of those halves of a word of two 16-bit floats that are infinite or NaN (all ones in the exponent), and all
// bits of such halves.
template <typename T>
__device__ __forceinline__ uint32_t odd_tops(uint32_t v) {
    constexpr uint32_t kExp = __is_same(T, __half) ? 0x7c007c00u : 0x7f807f80u, kOne = __is_same(T, __half) ? 0x04000400u : 0x00800080u;
    return ((v & kExp) + kOne) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t odd_halves(uint32_t v) {
    const uint32_t top = odd_tops<T>(v);
    return (top & 0x8000u ? 0xffffu : 0u) | (top >> 31 ? 0xffff0000u : 0u);
}

// Slots s0 .. s0 + 63 of a value tile (its rows from `at`) that are hidden from some row: those that nobody sees become 0,
// infinite and NaN elements of the others too, noted in *odd. By the 128 threads of a sub-tile, t of them.
template <typename T, int D>
__device__ __forceinline__ void clean_values(const Unit& u, uint8_t* at, int s0, int t, volatile int* odd) {
    constexpr int kPieces = D / 16;   // a thread's, half a row
    const int e = t & 63, s = s0 + e, first = (t >> 6) * kPieces;
    if (!hidden(u, s)) return;
    const bool dead = s >= u.hi || (s < u.lo && s >= u.sink);
    uint8_t* const row = at + e * 128;
    const auto piece = [&](int i) {
        return reinterpret_cast<uint4*>(row + ((first + i) >> 3) * Cut<D>::kBand + ((((first + i) ^ e) & 7) << 4));
    };
    if (dead) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) *piece(i) = make_uint4(0, 0, 0, 0);
        return;
    }
    uint32_t most[2] = {0, 0};   // of all 16-bit magnitudes, by halves
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const uint4 w = *piece(i);
        most[0] = __vmaxu2(most[0], w.x & 0x7fff7fffu), most[1] = __vmaxu2(most[1], w.y & 0x7fff7fffu);
        most[0] = __vmaxu2(most[0], w.z & 0x7fff7fffu), most[1] = __vmaxu2(most[1], w.w & 0x7fff7fffu);
    }
    if (!odd_tops<T>(__vmaxu2(most[0], most[1]))) return;
    *odd = 1;
    __threadfence_block();   // whoever finds the zeros finds the note
    for (int i = 0; i < kPieces; ++i) {
        uint4 w = *piece(i);
        w.x &= ~odd_halves<T>(w.x), w.y &= ~odd_halves<T>(w.y), w.z &= ~odd_halves<T>(w.z), w.w &= ~odd_halves<T>(w.w);
        *piece(i) = w;
    }
}

// What clean_values took out, back into row f's results of dims d .. d + N - 1: the sum of a row that sees an infinity or NaN.
template <typename T, int D, int N>
__device__ __noinline__ void add_odd(const Paged& c, const TileParams& p, const Unit& u, int f, int d, float (&o)[N]) {
    const int32_t* const table = table_of(c, p, u);
    const Sees sees(p, u, f);
    for (int k = u.c0; k < u.c1; ++k) {
        const int s0 = block_of(u, k) * Cut<D>::kKeys;
        if (!any_hidden<D>(u, s0, Cut<D>::kKeys)) continue;
        for (int s = s0; s < s0 + Cut<D>::kKeys; ++s) {
            if (!hidden(u, s) || !sees(s)) continue;
            const int id = table[s >> c.shift];
            if (!c.is_page(id)) continue;
            const T* const v = static_cast<const T*>(c.v) + c.row(id, u.hk, s) + d;
            for (int e = 0; e < N; ++e) {
                const float x = static_cast<float>(v[e]);
                if (!(x - x == 0.0f)) o[e] += x;
            }
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(Cut<D>::kThreads, 1)
    attn_tiles(const __grid_constant__ Paged c, const __grid_constant__ TileParams p, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap q_map,
               const __grid_constant__ CUtensorMap q_few_map) {
    using C = Cut<D>;
    constexpr bool kBf16 = !__is_same(T, __half);
    constexpr uint32_t kIdS = idesc(64, kBf16, false), kIdO = idesc(D, kBf16, true);
    // P is 2^(s - m + kUp): 16-bit floats of 5 exponent bits keep small ones so; with kSlack it stays below 2^15
    constexpr float kUp = kBf16 ? 0.0f : 8.0f;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared<C::kStages> sh;
    const uint32_t smem = (fer::dev::smem_addr(smem_raw) + 1023u) & ~1023u, ring = smem + C::kRing;
    uint8_t* const smem_at = smem_raw + (smem - fer::dev::smem_addr(smem_raw));
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;

    if (t == 0) {
        for (int i = 0; i < C::kStages; ++i) fer::dev::mbar_init(&sh.full[i], 1), fer::dev::mbar_init(&sh.empty[i], C::kSubs);
        for (int i = 0; i < kUnitSlots; ++i)
            fer::dev::mbar_init(&sh.unit_full[i], 1), fer::dev::mbar_init(&sh.unit_empty[i], C::kSoft + C::kSubs + 1);
        for (int i = 0; i < 2; ++i) fer::dev::mbar_init(&sh.q_full[i], 1), fer::dev::mbar_init(&sh.q_empty[i], C::kSubs);
        for (int i = 0; i < 2; ++i) {
            for (int j = 0; j < 2; ++j)
                fer::dev::mbar_init(&sh.s_full[i][j], 1), fer::dev::mbar_init(&sh.p_full[i][j], 4),
                    fer::dev::mbar_init(&sh.o_full[i][j], 1);
        }
        sh.stop = 0;
        sh.odd[0] = sh.odd[1] = 0;
        fer::dev::fence_mbar_init();
        fer::dev::prefetch_tmap(&k_map);
        fer::dev::prefetch_tmap(&v_map);
        if (p.q_maps != kQLoads) fer::dev::prefetch_tmap(&q_map);
        if (p.q_maps == kQBoxes) fer::dev::prefetch_tmap(&q_few_map);
    }
    if (w == C::kSoft + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fer::dev::smem_addr(&sh.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fer::dev::pdl_begin();

    // units before every segment of sequences
    const Prefix<D> pre(c, p);
    int seg = 1, segments = 1;
    if (alike(p)) {
        if (t == 0) {
            sh.sum[0] = p.own_chunk_log2 >= 0 ? 0 : p.n_seq * c.kv_heads * ((p.group - 1) / C::kRows + 1);
            if (pre.bad && blockIdx.x == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
        }
    } else {
        seg = (p.n_seq + kSegments - 1) / kSegments, segments = (p.n_seq + seg - 1) / seg;
        int mine[(kSegments + C::kThreads - 1) / C::kThreads] = {};
        bool bad = pre.bad, broken = false;
        int carry = 0;
        for (int k = 0, s0 = 0; s0 < segments; ++k, s0 += C::kThreads) {
            const int s = s0 + t;
            int n = 0;
            if (s < segments)
                for (int b = s * seg; b < min(p.n_seq, (s + 1) * seg); ++b) {
                    const Seq q(c, p, b);
                    bad = bad || q.bad;
                    broken = broken || q.broken;
                    if (!q.broken) n += units_of<D>(p, q) * c.kv_heads;
                }
            mine[k] = n;
            int x = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, off);
                if (lane >= off) x += y;
            }
            if (lane == 31) sh.sum[w] = x;
            __syncthreads();
            x += carry - n;
            for (int i = 0; i < C::kThreads / 32; ++i) {
                if (i < w) x += sh.sum[i];
                carry += sh.sum[i];
            }
            if (s < segments) sh.units[s] = x;
            __syncthreads();
        }
        // with offsets that cannot be nothing is done, here or by the joining
        broken = __syncthreads_or(broken);
        if (t == 0) {
            sh.sum[0] = broken ? 0 : carry;
            if (p.broken && blockIdx.x == 0) *p.broken = broken;
        }
        if ((bad || broken) && blockIdx.x == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const int units = sh.sum[0] + pre.units(c), grid = static_cast<int>(gridDim.x);
    const uint32_t tmem = sh.tmem;
    volatile int* const stop = &sh.stop;
    bool ok = true;

    if (w >= C::kSoft) {
        if constexpr (C::kShift) fewer_registers();   // all four warps of the group
        if (w == C::kSoft) {
            // ---- keys and values. Pages of a block: one a lane.
            const int box_rows = min(C::kKeys, c.page_size()), pages = C::kKeys / box_rows, boxes = pages * C::kBands;
            uint32_t tile = 0, block = 0;   // so far
            const auto take = [&](int k) {
                const int slot = k % kUnitSlots;
                if (ok) ok = warp_wait(&sh.unit_full[slot], k / kUnitSlots);
                Unit u = sh.unit[slot];
                __syncwarp();
                if (lane == 0) fer::dev::mbar_arrive(&sh.unit_empty[slot]);
                if (!ok || fer::dev::warp_flag(stop)) u.tok0 = -1;
                return u;
            };
            // this lane's page of block i of a unit: -1 where there is none to read
            const auto page_at = [&](const Unit& u, int i) {
                if (u.tok0 < 0 || i >= u.c1 - u.c0 || lane >= pages) return -1;
                const int page = ((block_of(u, u.c0 + i) * C::kKeys) >> c.shift) + lane;
                if (!page_needed(c, u, page)) return -1;
                const int id = table_of(c, p, u)[page];
                return id < 0 ? INT_MAX : id;   // out of range either way
            };
            Unit u = take(0);
            int id0 = page_at(u, 0), id1 = page_at(u, 1), id2 = page_at(u, 2);   // of blocks i, i + 1, i + 2
            for (int k = 0; ok && u.tok0 >= 0; ++k) {
                const int nb = u.c1 - u.c0, lead = loads_two<D>(u) ? 2 : 1;
                const auto load = [&](int i, int mine, bool value) {
                    const int st = tile % C::kStages;
                    if (ok) ok = warp_wait(&sh.empty[st], (tile / C::kStages & 1) ^ 1);
                    if (!ok) return;
                    const bool bad = __any_sync(0xffffffffu, mine >= c.pages);
                    if (lane == 0) {
                        if (!value) {
                            sh.bad[block % kBadRing] = bad;
                            if (bad) fer::dev::report(p.err, fer::dev::kErrBadShape);
                        }
                        fer::dev::mbar_arrive_expect_tx(&sh.full[st], C::kTile);
                    }
                    __syncwarp();
                    const int s0 = block_of(u, u.c0 + i) * C::kKeys;
                    for (int j0 = 0; j0 < boxes; j0 += 32) {
                        const int j = j0 + lane, pg = j / C::kBands, band = j % C::kBands;
                        const int id = __shfl_sync(0xffffffffu, mine, pg & 31);
                        // slots of no page are read as page `pages`, outside the map: zeros
                        if (j < boxes)
                            load_box(ring + st * C::kTile + band * C::kBand + pg * box_rows * 128, value ? &v_map : &k_map,
                                     band * 64, s0 & (c.page_size() - 1), u.hk, c.is_page(id) ? id : c.pages, &sh.full[st]);
                    }
                    ++tile;
                    if (!value) ++block;
                };
                if (nb > 0) load(0, id0, false);
                if (lead == 2 && nb > 1) load(1, id1, false);
                // the next unit's first ids are on their way while this one's last tiles wait for room
                Unit next{};
                int n0 = -1, n1 = -1, n2 = -1;
                for (int i = 0; i < max(nb, 1) && ok; ++i) {
                    const int id3 = page_at(u, i + 3);
                    if (i + 1 >= nb && u.last) {
                        next.tok0 = -1;
                    } else if (i + 1 >= nb) {
                        next = take(k + 1);
                        n0 = page_at(next, 0), n1 = page_at(next, 1), n2 = page_at(next, 2);
                    }
                    if (nb > 0) load(i, id0, true);
                    if (i + lead < nb) load(i + lead, lead == 2 ? id2 : id1, false);
                    id0 = id1, id1 = id2, id2 = id3;
                }
                u = next;
                id0 = n0, id1 = n1, id2 = n2;
            }
            if (!ok) {
                if (lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutSync);
                *stop = 1;
            }
            // the copies have landed before this warp leaves, whatever became of the others
            for (uint32_t i = tile > C::kStages ? tile - C::kStages : 0; i < tile; ++i)
                if (!warp_wait(&sh.full[i % C::kStages], i / C::kStages)) {
                    if (lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutLoad);
                    *stop = 1;
                }
        } else if (w > C::kSoft && w <= C::kSoft + C::kSubs) {
            // ---- products of sub-tile x. Each of these warps sees every tile of the ring, so that none can lap it, and lets go
            // of those that are the other's as soon as they are there.
            const int x = uniform(w - C::kSoft - 1);
            const uint32_t s_at = uniform(tmem) + 128 * x, o_at = uniform(tmem) + C::kColO + x * D;
            uint32_t tile = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0}, n_o = 0;   // so far
            int turn = 0;   // whose place among the queries the next unit of one sub-tile takes
            const auto landed = [&](uint32_t i) {
                if (ok) ok = warp_wait(&sh.full[i % C::kStages], i / C::kStages);
            };
            const auto skip = [&]() {
                landed(tile);
                if (lane == 0) fer::dev::mbar_arrive(&sh.empty[tile % C::kStages]);
                ++tile;
            };
            for (int k = 0; ok; ++k) {
                const int slot = k % kUnitSlots;
                ok = warp_wait(&sh.unit_full[slot], k / kUnitSlots);
                if (!ok || fer::dev::warp_flag(stop)) break;
                const int nf = uniform(sh.unit[slot].nf), nb = uniform(sh.unit[slot].c1 - sh.unit[slot].c0);
                const bool end = uniform(sh.unit[slot].tok0) < 0, last = uniform(sh.unit[slot].last) != 0;
                __syncwarp();
                if (lane == 0) fer::dev::mbar_arrive(&sh.unit_empty[slot]);
                if (end) break;
                if (nb == 0) {
                    if (last) break;
                    continue;
                }
                const bool alt = C::kSubs == 2 && nf <= 128, fine = nf <= C::kFine && nf > kFew;
                // a unit of one sub-tile has one place, they take turns; else each sub-tile has its own
                const int q_at = C::kSubs == 1 ? 0 : alt ? turn : x;
                const uint32_t q_desc = desc_low(smem + q_at * C::kQ, 16);
#pragma unroll
                for (int i = 0; i < C::kSubs; ++i)
                    if (!alt || i == q_at) ok = ok && warp_wait(&sh.q_full[i], n_q[i]++);
                if (C::kSubs == 2 && !alt && lane == 0) fer::dev::mbar_arrive(&sh.q_empty[x ^ 1]);   // not read here
                if (alt) turn ^= 1;
                // S of 64 keys of tile i, and O += P V of 64
                const auto product_s = [&](uint32_t i, int h, int at) {
                    const uint32_t kk = desc_low(ring + i % C::kStages * C::kTile + h * 8192, 16);
#pragma unroll
                    for (int j = 0; j < D / 16; ++j)
                        mma_ss(s_at + 64 * at, q_desc + ((j / 4) * 16384 + (j % 4) * 32) / 16,
                               kk + ((j / 4) * C::kBand + (j % 4) * 32) / 16, kIdS, j > 0);
                    commit(&sh.s_full[x][at]);
                };
                const auto product_o = [&](uint32_t i, int h, int at, bool first) {
                    const uint32_t v = desc_low(ring + i % C::kStages * C::kTile + h * 8192, C::kBand);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_ts(o_at, s_at + 64 * at + 32 * (j >> 1) + 8 * (j & 1), v + j * (2048 / 16), kIdO, !first || j > 0);
                    if (fine)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma_ts(o_at, s_at + 64 * at + 32 * (j >> 1) + 16 + 8 * (j & 1), v + j * (2048 / 16), kIdO, 1);
                    commit(&sh.o_full[x][n_o & 1]);
                };
                // the tile's last reader lets go of it
                const auto done = [&](uint32_t i) { commit(&sh.empty[i % C::kStages]); };
                const auto given = [&](int at) {
                    if (ok) ok = warp_wait(&sh.p_full[x][at], n_p[at]);
                    ++n_p[at];
                    fence_after();
                };
                if constexpr (C::kSubs == 1) {
                    // K_0 K_1 V_0 K_2 V_1 ...: a block is 64 keys, and S of the next but one follows
                    for (int i = 0; i < min(nb, 2); ++i) {
                        landed(tile);
                        fence_after();
                        if (ok && elected()) {
                            product_s(tile, 0, i);
                            done(tile);
                            if (i + 1 == nb) commit(&sh.q_empty[q_at]);
                        }
                        __syncwarp();
                        ++tile;
                    }
                    for (int i = 0; i < nb; ++i) {
                        const bool more = i + 2 < nb;
                        landed(tile);
                        if (more) landed(tile + 1);
                        given(i & 1);
                        if (ok && elected()) {
                            product_o(tile, 0, i & 1, i == 0);
                            done(tile);
                            if (more) {
                                product_s(tile + 1, 0, i & 1);
                                done(tile + 1);
                                if (i + 3 == nb) commit(&sh.q_empty[q_at]);
                            }
                        }
                        __syncwarp();
                        ++n_o;
                        tile += more ? 2 : 1;
                    }
                } else {
                    // K_0 V_0 K_1 V_1 ..., or K_0 K_1 V_0 K_2 V_1 ... where even blocks are sub-tile 0's: either way the values
                    // of a block are followed by the keys of this sub-tile's next
                    const int step = alt ? 2 : 1;
                    if (alt && x == 1) skip();                                   // K_0
                    if (alt && x == 1 && nb == 1) {
                        skip();                                                  // V_0
                        if (lane == 0) fer::dev::mbar_arrive(&sh.q_empty[q_at]);
                        if (last) break;
                        continue;
                    }
                    landed(tile);
                    fence_after();
                    if (ok && elected()) {
                        product_s(tile, 0, 0);
                        product_s(tile, 1, 1);
                        done(tile);
                        if (step >= nb - (alt ? x : 0)) commit(&sh.q_empty[q_at]);
                    }
                    __syncwarp();
                    ++tile;
                    if (alt && x == 0 && nb > 1) skip();                         // K_1
                    for (int i = alt ? x : 0; i < nb; i += step) {
                        if (alt && i > 0) {
                            skip();                                              // the other's V_{i-1}
                            if (i + 1 < nb) skip();                              // and K_{i+1}
                        }
                        const bool more = i + step < nb;
                        landed(tile);
                        if (more) landed(tile + 1);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            given(h);
                            if (ok && elected()) {
                                product_o(tile, h, h, h == 0 && i < step);
                                if (h == 1) done(tile);
                                if (more) {
                                    product_s(tile + 1, h, h);
                                    if (h == 1) {
                                        done(tile + 1);
                                        if (i + 2 * step >= nb) commit(&sh.q_empty[q_at]);
                                    }
                                }
                            }
                            __syncwarp();
                            ++n_o;
                        }
                        tile += more ? 2 : 1;
                    }
                    if (alt && (nb - 1) % 2 != x) skip();                        // the other's last values
                }
                if (last) break;
            }
            if (!ok) {
                if (lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutLoad);
                *stop = 1;
            }
        } else {
            // ---- units, one ahead, and their queries, read while the unit before still computes; few rows go to each quarter of
            // the sub-tile
            uint32_t n_q[2] = {0, 0};
            int turn = 0;
            const auto publish = [&](int k) {
                const int slot = k % kUnitSlots;
                if (ok) ok = warp_wait(&sh.unit_empty[slot], (k / kUnitSlots & 1) ^ 1);
                const long long x = static_cast<long long>(k) * grid + (k & 1 ? grid - 1 - blockIdx.x : blockIdx.x);
                Unit u{};
                u.tok0 = -1;
                if (!ok || fer::dev::warp_flag(stop)) return u;
                bool bad = false;
                if (x < units) u = find_unit<D>(c, p, pre, sh.units, segments, seg, static_cast<int>(x), bad);
                // the next round's is one of the next grid's
                u.last = static_cast<long long>(k + 1) * grid + (k & 1 ? blockIdx.x : grid - 1 - blockIdx.x) >= units;
                if (lane == 0) {
                    if (bad) fer::dev::report(p.err, fer::dev::kErrBadShape);
                    sh.unit[slot] = u;
                    fer::dev::mbar_arrive(&sh.unit_full[slot]);
                }
                __syncwarp();
                return u;   // the last: a later round has none either
            };
            const auto queries = [&](const Unit& u) {
                if (u.c1 == u.c0) return;
                const bool alt = alternate<D>(u);
                const int copies = u.nf <= kFew ? 4 : 1;
#pragma unroll
                for (int i = 0; i < C::kSubs; ++i) {
                    if (alt && i != turn) continue;
                    ok = ok && warp_wait(&sh.q_empty[i], n_q[i]++ ^ 1u);   // what was there has been multiplied
                    if (!ok) break;
                    const int f0 = u.f0 + (alt ? 0 : 128 * i), rows = min(128, u.f0 + u.nf - f0);
                    const uint32_t to = smem + i * C::kQ;
                    if (p.q_maps == kQBoxes) {
                        // all rows, or a quarter's for each, in one box a band: rows behind the unit's are of no matter
                        if (lane == 0) fer::dev::mbar_arrive_expect_tx(&sh.q_full[i], C::kQ);
                        __syncwarp();
                        if (lane < copies * C::kBands)
                            load_q(to + lane % C::kBands * 16384 + lane / C::kBands * 4096, copies == 1 ? &q_map : &q_few_map,
                                   lane % C::kBands * 64, u.hk * p.group, u.tok0 + p.by_group(f0), &sh.q_full[i]);
                    } else if (p.q_maps == kQRows) {
                        if (lane == 0) fer::dev::mbar_arrive_expect_tx(&sh.q_full[i], rows * copies * C::kBands * 128);
                        __syncwarp();
                        for (int j = lane; j < rows * copies; j += 32) {
                            const int f = copies == 1 ? j : j >> 2, row = copies == 1 ? j : f + 32 * (j & 3);
                            const int tok = p.by_group(f0 + f), g = f0 + f - tok * p.group;
                            for (int band = 0; band < C::kBands; ++band)
                                load_q(to + band * 16384 + row * 128, &q_map, band * 64, u.hk * p.group + g, u.tok0 + tok, &sh.q_full[i]);
                        }
                    } else {
                        // rows at addresses that tensor copies do not take
                        for (int j = lane; j < rows * (D / 8); j += 32) {
                            const int f = j / (D / 8), pc = j % (D / 8), tok = p.by_group(f0 + f), g = f0 + f - tok * p.group;
                            const uint16_t* const src = reinterpret_cast<const uint16_t*>(p.q) + (static_cast<size_t>(u.tok0) + tok) * p.qs +
                                                        (static_cast<size_t>(u.hk) * p.group + g) * D + pc * 8;
                            uint32_t e[4];
#pragma unroll
                            for (int h = 0; h < 4; ++h) e[h] = src[2 * h] | static_cast<uint32_t>(src[2 * h + 1]) << 16;
                            for (int c4 = 0; c4 < copies; ++c4)
                                *reinterpret_cast<uint4*>(smem_at + i * C::kQ + (pc >> 3) * 16384 + (f + 32 * c4) * 128 +
                                                          (((pc ^ f) & 7) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
                        }
                        fer::dev::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) fer::dev::mbar_arrive(&sh.q_full[i]);
                    }
                    __syncwarp();
                }
                if (alt) turn ^= 1;
            };
            Unit u = publish(0);
            if (u.tok0 >= 0) {
                queries(u);
                if (u.last) u.tok0 = -1;
                else u = publish(1);
            }
            for (int k = 1; ok && u.tok0 >= 0; ++k) {
                Unit next = u;
                next.tok0 = -1;
                if (!u.last) next = publish(k + 1);
                queries(u);
                u = next;
            }
            // the copies have landed before this warp leaves, whatever became of the others
#pragma unroll
            for (int i = 0; i < C::kSubs; ++i)
                if (p.q_maps != kQLoads && n_q[i] > 0 && ok) ok = warp_wait(&sh.q_full[i], n_q[i] - 1);
            if (!ok) {
                if (lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutSync);
                *stop = 1;
            }
        }
    } else {
        // ---- softmax, a row a thread, 64 keys at a time; of few rows (kFew) each is in all four quarters of a sub-tile: two take
        // the first and two the second 32 keys, and of each two one keeps P's upper and one its lower 16 bits
        if constexpr (C::kShift) more_registers();
        const int x = w >> 2, r = t & 127, half = (w >> 1) & 1, part = w & 1;
        const uint32_t row_at = tmem + (static_cast<uint32_t>((w & 3) * 32) << 16);
        uint32_t base = 0, block = 0, n_s0 = 0, n_s1 = 0, n_o = 0;   // n_o: P given so far
        for (int k = 0;; ++k) {
            const int slot = k % kUnitSlots;
            ok = ok && warp_wait(&sh.unit_full[slot], k / kUnitSlots);
            // both sub-tiles' warps leave together: each unit has barriers for all of them
            if (!ok) *stop = 1;
            // and the unit before is done with its sums and results
            const bool leave = meet_or<32 * C::kSoft>(!ok || *stop);
            volatile int* const odd_here = &sh.odd[k & 1];
            if (t == 0) sh.odd[(k + 1) & 1] = 0;
            if (leave) {
                if (!ok && lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutMma);
                break;
            }
            const Unit u = sh.unit[slot];
            __syncwarp();
            if (lane == 0) fer::dev::mbar_arrive(&sh.unit_empty[slot]);
            if (u.tok0 < 0) break;
            const int nb = u.c1 - u.c0, nf = u.nf;
            const bool alt = alternate<D>(u), few = nf <= kFew, fine = nf <= C::kFine;
            const int f = few ? lane : alt ? r : x * 128 + r, first = alt ? x : 0, step = alt ? 2 : 1;
            const bool rows_here = (f & ~31) < nf;                         // of the warp
            const bool real = f < nf;                                      // rows behind the unit's hold anything
            const Sees sees(p, u, min(f, nf - 1));
            // what every row of the warp sees, for blocks that need no mask
            const int all_end = __reduce_min_sync(0xffffffffu, sees.end), all_begin = __reduce_max_sync(0xffffffffu, sees.begin);
            float m = -INFINITY, l = 0.0f;

            // The products given so far have been added. They take turns at two barriers: where S of 64 keys is there, the
            // products of all but the 64 before them are.
            const auto o_added = [&]() { return warp_wait(&sh.o_full[x][(n_o - 1) & 1], (n_o - 1) >> 1); };
            // The blocks, 64 keys at a time, N chunks of 32 of them from chunk j0 on. kind 0: P is rounded, 1: what that leaves is
            // kept too, 2: one of the two for these keys, and 0 for the others. P of a chunk lies over its own scores: 16 words,
            // and what is left behind them. The next scores are on their way while P is handed over.
            // Where both sub-tiles have rows of their own their exponentials take turns, so that one's are computed while the
            // other's scores and products are on their way: left alone the two fall into step (a long causal piece 2028 us without turns, 1958 with).
            const auto my_turn = [&]() { if (C::kSubs == 2 && !alt) asm volatile("bar.sync %0, 256;" ::"r"(2 + x) : "memory"); };
            const auto your_turn = [&]() { if (C::kSubs == 2 && !alt) asm volatile("bar.arrive %0, 256;" ::"r"(3 - x) : "memory"); };
            if (!alt && nb > 0 && x == 1) your_turn();
            const auto blocks = [&](auto chunks, auto kind, int j0) {
                constexpr int N = decltype(chunks)::value, kKind = decltype(kind)::value;
                float v[N][32];
                const auto load = [&](int at) {   // scores of 64 keys, when they are there
                    if (ok) ok = warp_wait(&sh.s_full[x][at], at ? n_s1 : n_s0);
                    at ? ++n_s1 : ++n_s0;
                    fence_after();
#pragma unroll
                    for (int j = 0; j < N; ++j) tmem_ld(row_at + 128 * x + 64 * at + 32 * (j0 + j), v[j]);
                };
                const auto hand_over = [&](int at) {
                    fence_before();
                    __syncwarp();
                    if (lane == 0) fer::dev::mbar_arrive(&sh.p_full[x][at]);
                    ++n_o;
                };
                int i = first, h = 0;
                load(C::kParts == 1 ? i & 1 : 0);
                wait_ld(v);
#pragma unroll 1
                for (;;) {
                    const int at = C::kParts == 1 ? i & 1 : h, s0 = block_of(u, u.c0 + i) * C::kKeys + 64 * h;
                    const uint32_t s_at = row_at + 128 * x + 64 * at;
                    {
                        const bool bad = sh.bad[(block + i) % kBadRing] != 0;
                        if (bad || s0 + 64 > all_end || (s0 < all_begin && s0 + 64 > sees.sink)) {
#pragma unroll
                            for (int j = 0; j < N; ++j) {
                                // [begin, end) of the window and [0, sink) within the chunk
                                const int s1 = s0 + 32 * (j0 + j);
                                uint32_t on = (below(sees.end - s1) & ~below(sees.begin - s1)) | below(min(sees.sink, sees.end) - s1);
                                if (bad)
                                    for (int e = 0; e < 32; e += 8) {   // pages are of 8 slots and more
                                        const int page = (s1 + e) >> c.shift;
                                        if (!page_needed(c, u, page) || !c.is_page(table_of(c, p, u)[page])) on &= ~(0xffu << e);
                                    }
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (!(on >> e & 1u)) v[j][e] = -INFINITY;
                            }
                        }
                        float mx[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
#pragma unroll
                        for (int e = 4; e < 32 * N; e += 2)
                            mx[(e >> 1) & 3] = max3f(mx[(e >> 1) & 3], v[e >> 5][e & 31], v[e >> 5][(e & 31) + 1]);
                        // a score of +inf or NaN makes the row NaN: by its maximum, as powers2 does not hand a NaN on
                        float top = max3f(max3f(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale2;
                        if (top == INFINITY) top = NAN;
                        const bool raise = real && !(top <= m + kSlack);
                        if (__any_sync(0xffffffffu, raise)) {
                            const float m1 = raise ? top : m, a = raise ? ex2(m - m1) : 1.0f;   // 0 while m is -inf
                            m = m1;
                            l *= a;
                            if (i > first || h > 0) {
                                if (ok) ok = o_added();
                                fence_after();
#pragma unroll 1
                                for (int j = 0; j < D / 16; ++j) {
                                    uint32_t o[16];
                                    tmem_ld16(row_at + C::kColO + x * D + 16 * j, o);
#pragma unroll
                                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
                                    tmem_st16(row_at + C::kColO + x * D + 16 * j, o);
                                }
                            }
                        }
                        if (kKind == 0) my_turn();
                        const uint64_t sc2 = fer::dev::f2_splat(p.scale2), nm2 = fer::dev::f2_splat(kUp - (m == -INFINITY ? 0.0f : m));
                        uint64_t sum[2] = {0, 0};
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            uint32_t hi[16], low[16];
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                float p0, p1;
                                const uint64_t t2 = fer::dev::f2_fma(fer::dev::f2_pack(v[j][e], v[j][e + 1]), sc2, nm2);
                                if (kKind == 0 && (e >> 1) % kPolyOf < kPoly) {
                                    powers2(t2, p0, p1);
                                } else {
                                    fer::dev::f2_unpack(t2, p0, p1);
                                    p0 = ex2(p0), p1 = ex2(p1);
                                }
                                sum[(e >> 1) & 1] = fer::dev::f2_add(sum[(e >> 1) & 1], fer::dev::f2_pack(p0, p1));
                                hi[e >> 1] = pack2<T>(p0, p1);
                                if constexpr (kKind > 0) {
                                    float h0, h1;
                                    unpack2<T>(hi[e >> 1], h0, h1);
                                    low[e >> 1] = pack2<T>(p0 - h0, p1 - h1);
                                    if (kKind == 2) hi[e >> 1] = part ? low[e >> 1] : hi[e >> 1], low[e >> 1] = 0;
                                }
                            }
                            tmem_st16(s_at + 32 * (j0 + j), hi);
                            if constexpr (kKind > 0) tmem_st16(kKind == 1 ? s_at + 32 * j + 16 : s_at + 32 * (1 - j0), low);
                        }
                        if (kKind == 0 && (x == 0 || i + 1 < nb || h + 1 < C::kParts)) your_turn();
                        float sm[4];
                        fer::dev::f2_unpack(sum[0], sm[0], sm[1]);
                        fer::dev::f2_unpack(sum[1], sm[2], sm[3]);
                        l += (sm[0] + sm[1]) + (sm[2] + sm[3]);
                    }
                    if (any_hidden<D>(u, s0, 64) && ok) {
                        const uint32_t tile = base + at_v(loads_two<D>(u), i, nb);
                        ok = warp_wait(&sh.full[tile % C::kStages], tile / C::kStages);
                        if (ok) clean_values<T, D>(u, smem_at + C::kRing + tile % C::kStages * C::kTile + h * 8192, s0, r, odd_here);
                        fer::dev::fence_proxy_async_smem();
                    }
                    if (++h == C::kParts) h = 0, i += step;
                    if (i >= nb) {
                        wait_st();
                        hand_over(at);
                        break;
                    }
                    // S of the next 64 keys lies elsewhere, and has been on its way since P before this was handed over
                    load(C::kParts == 1 ? i & 1 : h);
                    wait_st();
                    hand_over(at);
                    wait_ld(v);
                }
            };
            if (first < nb) {
                using Zero = std::integral_constant<int, 0>;
                using One = std::integral_constant<int, 1>;
                using Two = std::integral_constant<int, 2>;
                if (few) blocks(One{}, Two{}, half);
                else if (fine) blocks(Two{}, One{}, 0);
                else blocks(Two{}, Zero{}, 0);
            }
            const bool mine = first < nb;
            if (mine && ok) ok = o_added();
            fence_after();
            base += 2 * nb, block += nb;

            // The results. Where blocks alternate, or rows are in several quarters, a row's sums meet first; everything stops
            // at the next unit where a wait ran out.
            float2* const sums = reinterpret_cast<float2*>(smem_at + C::kMeet);
            const uint32_t o_at = row_at + C::kColO + x * D;
            if (few) {
                constexpr int kParts = 4 * C::kSubs;   // sums of a row; m and l are those of half of them
                sums[t] = make_float2(m, l);
                meet<32 * C::kSoft>();
                float all = -INFINITY, total = 0.0f;
#pragma unroll
                for (int i = 0; i < kParts; i += 2) all = fmaxf(all, sums[32 * i + lane].x);
                const float base2 = all == -INFINITY ? 0.0f : all;
#pragma unroll
                for (int i = 0; i < kParts; i += 2) total = fmaf(sums[32 * i + lane].y, ex2(sums[32 * i + lane].x - base2), total);
                const float scale = u.part >= 0 ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
                const float mine2 = mine && ok ? ex2(m - base2) * scale : 0.0f;
                meet<32 * C::kSoft>();                 // the sums have been read
                const bool on = lane < nf;
                if (w == 0 && on) {
                    const size_t bh = q_row(p, u, lane) * p.heads + q_head(p, u, lane);
                    if (u.part >= 0) *reinterpret_cast<float2*>(p.part_ml + 2 * (bh * p.parts + u.part)) = make_float2(all, total);
                    else if (p.lse) p.lse[bh] = total == 0.0f ? -INFINITY : (all + (log2f(total) - kUp)) * kLn2;
                }
                // as many dims at once as there is room for: 4 KB a warp
                const int width = min(D, nf <= 8 ? 128 : nf <= 16 ? 64 : 32), rows = 1024 / width;
                float* const meet_at = reinterpret_cast<float*>(smem_at + C::kMeet);
                // the dims of this warp from d + e0 on, several loads under way at once
                const auto gather = [&](auto loads, int d, int e0) {
                    constexpr int N = decltype(loads)::value;
                    float o[N][32];
#pragma unroll
                    for (int j = 0; j < N; ++j) tmem_ld(o_at + d + e0 + 32 * j, o[j]);   // without sums: anything
                    wait_ld(o);
                    if (on) {
#pragma unroll
                        for (int e = 0; e < 32 * N; e += 4) {
                            // 16-byte pieces of neighbouring rows in different banks
                            float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            const float* const from = o[e >> 5] + (e & 31);
                            if (mine && ok) q = make_float4(from[0] * mine2, from[1] * mine2, from[2] * mine2, from[3] * mine2);
                            *reinterpret_cast<float4*>(meet_at + (w * rows + lane) * width + e0 + (e & ~31) + ((e ^ (lane << 2)) & 28)) = q;
                        }
                    }
                    __syncwarp();
                };
                const bool odd = *odd_here != 0;
                for (int d = 0; d < D; d += width) {
                    if (width == 32) gather(std::integral_constant<int, 1>{}, d, 0);
                    else
                        for (int e0 = 0; e0 < width; e0 += 64) gather(std::integral_constant<int, 2>{}, d, e0);
                    meet<32 * C::kSoft>();
                    for (int i = t; i < nf * width; i += 32 * C::kSoft) {
                        const int row = i / width, e = i % width;
                        const float* const from = meet_at + row * width + (e & ~31) + (((e ^ (row << 2)) & 28) | (e & 3));
                        float v = 0.0f;
#pragma unroll
                        for (int g = 0; g < kParts; ++g) v += from[g * rows * width];
                        if (nb == 0) v = 0.0f;
                        if (odd) {
                            float one[1] = {v};
                            add_odd<T, D, 1>(c, p, u, row, d + e, one);
                            v = one[0];
                        }
                        const size_t tok = q_row(p, u, row);
                        const int head = q_head(p, u, row);
                        if (u.part >= 0) p.part_o[((tok * p.heads + head) * p.parts + u.part) * D + d + e] = v;
                        else put(static_cast<T*>(p.out) + tok * p.os + static_cast<size_t>(head) * D + d + e, v);
                    }
                    meet<32 * C::kSoft>();
                }
            } else {
                float all = m, wa = 1.0f, wb = 0.0f, total = l;
                uint32_t at_a = o_at, at_b = o_at;
                int d0 = 0, d1 = D;
                if (alt) {   // each sub-tile's warps take half of the dims of both sums
                    sums[t] = make_float2(m, l);
                    meet<32 * C::kSoft>();
                    const float2 sa = sums[r], sb = sums[128 + r];
                    all = fmaxf(sa.x, sb.x);
                    const float base2 = all == -INFINITY ? 0.0f : all;
                    wa = ex2(sa.x - base2), wb = ex2(sb.x - base2);
                    total = sa.y * wa + sb.y * wb;
                    meet<32 * C::kSoft>();   // the sums have been read
                    d0 = x * (D / 2), d1 = d0 + D / 2;
                    at_a = row_at + C::kColO, at_b = at_a + D;
                    fence_after();
                }
                const bool on = f < nf;
                const int fr = min(f, nf - 1), head = q_head(p, u, fr);
                const size_t tok = q_row(p, u, fr), bh = tok * p.heads + head, place = bh * p.parts + max(u.part, 0);
                const float scale = u.part >= 0 ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
                wa *= scale, wb *= scale;
                if (rows_here && ok) {
                    const bool odd = *odd_here != 0;
                    // 128 bytes of each of the warp's rows at a time, turned round in shared memory, so that eight lanes write a
                    // row's 128 bytes
                    uint8_t* const turn = smem_at + C::kMeet + w * 4096;
                    const unsigned long long to = u.part >= 0 ? reinterpret_cast<unsigned long long>(p.part_o + place * D)
                                                              : reinterpret_cast<unsigned long long>(static_cast<T*>(p.out) + tok * p.os + static_cast<size_t>(head) * D);
                    const bool whole = u.part >= 0 || (reinterpret_cast<uintptr_t>(p.out) | (p.os * 2)) % 16 == 0;
                    const int rows = min(32, nf - (f - lane)), size = u.part >= 0 ? 4 : 2;
                    uint8_t* const mine_at = turn + lane * 128;
                    const int span = u.part >= 0 ? 32 : 64;   // dims in 128 bytes
#pragma unroll 1
                    for (int d = d0; d < d1; d += 32) {
                        float o[32];
                        {
                            float a[2][32];
                            tmem_ld(at_a + d, a[0]);   // without sums: anything
                            tmem_ld(at_b + d, a[1]);
                            wait_ld(a);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                o[e] = nb > 0 ? a[0][e] * wa : 0.0f;
                                if (alt && nb > 1) o[e] = fmaf(a[1][e], wb, o[e]);
                            }
                        }
                        if (odd) {
                            float y[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) y[e] = o[e];
                            add_odd<T, D, 32>(c, p, u, fr, d, y);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = y[e];
                        }
                        const int off = (d - d0) % span;
                        if (u.part >= 0) {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                *reinterpret_cast<float4*>(mine_at + (((off / 4 + e) ^ lane) & 7) * 16) =
                                    make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                *reinterpret_cast<uint4*>(mine_at + (((off / 8 + e) ^ lane) & 7) * 16) =
                                    make_uint4(pack2<T>(o[8 * e], o[8 * e + 1]), pack2<T>(o[8 * e + 2], o[8 * e + 3]),
                                               pack2<T>(o[8 * e + 4], o[8 * e + 5]), pack2<T>(o[8 * e + 6], o[8 * e + 7]));
                        }
                        if (off + 32 < span && d + 32 < d1) continue;
                        __syncwarp();
                        const int begin = d - off, pieces = (off + 32) * size / 16;
                        const unsigned long long column = static_cast<unsigned long long>(begin) * size + (lane & 7) * 16;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const int row = i + (lane >> 3);
                            const unsigned long long at = __shfl_sync(0xffffffffu, to, row);
                            if (row < rows && (lane & 7) < pieces) {
                                const uint4 v = *reinterpret_cast<const uint4*>(turn + row * 128 + (((lane ^ row) & 7) << 4));
                                if (whole) {
                                    *reinterpret_cast<uint4*>(at + column) = v;
                                } else {
                                    uint16_t* const h = reinterpret_cast<uint16_t*>(at + column);
                                    h[0] = v.x, h[1] = v.x >> 16, h[2] = v.y, h[3] = v.y >> 16;
                                    h[4] = v.z, h[5] = v.z >> 16, h[6] = v.w, h[7] = v.w >> 16;
                                }
                            }
                        }
                        __syncwarp();
                    }
                    if (on && d0 == 0) {
                        if (u.part >= 0) *reinterpret_cast<float2*>(p.part_ml + 2 * place) = make_float2(all, total);
                        else if (p.lse) p.lse[bh] = total == 0.0f ? -INFINITY : (all + (log2f(total) - kUp)) * kLn2;
                    }
                }
            }
            fence_before();
            if (u.last) {
                if (!ok) {
                    *stop = 1;
                    if (lane == 0) fer::dev::report(p.err, fer::dev::kErrTimeoutMma);
                }
                break;
            }
        }
    }

    fence_before();
    __syncthreads();
    if (w == C::kSoft + 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Adds the parts of every row that has several, one warp each: out = sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m).
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) attn_join(const Paged c, const TileParams p, float up) {
    constexpr int kV = D / 32;
    struct alignas(4 * (kV < 4 ? kV : 4)) Dims { float e[kV]; };
    fer::dev::pdl_begin();
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);
    if (item >= static_cast<long long>(p.rows) * p.heads || (p.broken && *p.broken)) return;
    const int tok = static_cast<int>(item / p.heads), head = static_cast<int>(item - static_cast<long long>(tok) * p.heads);
    int own = 0, shared = 0;
    {
        // the row's sequence, and its tile's blocks
        int b = tok;
        if (p.offsets) {
            int lo = 0, hi = p.n_seq;   // the last sequence that starts at or before the row
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (p.offsets[mid] <= tok) lo = mid;
                else hi = mid;
            }
            b = lo;
        }
        const Seq q(c, p, b);
        if (tok < q.tok0 || tok >= q.tok0 + q.n) return;   // of no sequence
        const long long f = static_cast<long long>(tok - q.tok0) * p.group + head % p.group;
        Unit u;
        if (p.own_chunk_log2 >= 0) own = (q.len + (1 << p.own_chunk_log2) - 1) >> p.own_chunk_log2;
        else own = chunks_of(tile_range<D>(p, q, static_cast<int>(f / Cut<D>::kRows), u), p.chunk);
    }
    if (p.prefix_pages) shared = Prefix<D>(c, p).chunks;
    else if (own == 1) return;   // written already
    // the other kernel's parts are not 2^up times as large
    const bool other = p.own_chunk_log2 >= 0;
    const float2* const ml = reinterpret_cast<const float2*>(p.part_ml) + item * p.parts + (other ? 0 : p.own_parts);
    const float* const po = p.part_o + (item * p.parts + (other ? 0 : p.own_parts)) * D + kV * lane;
    const float2* const own_ml = other ? reinterpret_cast<const float2*>(p.own_ml) + item * p.own_parts : ml - p.own_parts;
    const float* const own_o = other ? p.own_o + item * p.own_parts * D + kV * lane : po - static_cast<size_t>(p.own_parts) * D;
    const float lift = other ? up : 0.0f;
    const auto part_ml = [&](int i) {
        float2 v = i < own ? own_ml[i] : ml[i - own];
        if (i < own) v.x += lift;
        return v;
    };
    const int n = own + shared;
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, part_ml(i).x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    Dims o{};
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        const float2 v = part_ml(i);
        const Dims d = *reinterpret_cast<const Dims*>(i < own ? own_o + static_cast<size_t>(i) * D : po + static_cast<size_t>(i - own) * D);
        const float y = ex2(v.x - base);
        l = fmaf(v.y, y, l);
        // a part without a key counts as nothing, and one that vanishes gives an infinite value its due
        const float z = v.y == 0.0f ? 0.0f : fmaxf(y, 1.17549435e-38f);
#pragma unroll
        for (int e = 0; e < kV; ++e) o.e[e] = fmaf(d.e[e], z, o.e[e]);
    }
    T* const out = static_cast<T*>(p.out) + static_cast<size_t>(tok) * p.os + static_cast<size_t>(head) * D + kV * lane;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < kV; ++e) put(out + e, l == 0.0f ? 0.0f : o.e[e] * inv);
    if (lane == 0 && p.lse) p.lse[item] = l == 0.0f ? -INFINITY : (base + (log2f(l) - up)) * kLn2;
}

// ---- host

struct Split {
    int chunk, parts;
};

constexpr int keys_of(int head_dim) { return head_dim == 256 ? 64 : 128; }
constexpr int rows_of(int head_dim) { return head_dim == 256 ? 128 : 256; }

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Into how many parts to cut `blocks` key blocks of each of `tiles` tiles: the number of at most `most` with which the GPU is
// done first, by the rounds of its SMs times the blocks of a part and what a unit costs beside them.
long long fewest_rounds(long long tiles, long long blocks, long long most) {
    long long best = 1, least = LLONG_MAX;
    for (long long parts = 1; parts <= most; ++parts) {
        const long long chunk = ceil_div(blocks, parts), units = tiles * ceil_div(blocks, chunk);
        const long long time = ceil_div(units, kSms) * (chunk + kUnitBlocks);
        if (time < least) least = time, best = parts;
    }
    return best;
}

// Cuts of a row's key blocks, of which there are at most `blocks`, where `units` tiles of rows and heads are to be
// shared out and a tile has about tile_rows rows. A tile of few rows is bound by HBM, and a part costs it what reading some
// 300 keys does, so cuts are for even shares: of 1024 keys or more where there are fewer tiles than SMs, else of 2560 (64
// sequences x 8 key heads behind a window of 2048: whole 146 us, in halves 158; over 8192 slots: whole 421, in parts 282).
Split split(long long units, long long blocks, long long tile_rows, int keys) {
    Split s{INT_MAX, 0};
    long long parts = 1;
    if (tile_rows <= 64) {
        const bool many = units >= kSms;
        const long long most = ceil_div((many ? 12 : 6) * kSms, units);
        parts = ceil_div(blocks, (many ? 2560 : 1024) / keys);
        if (parts > most) parts = most;
    } else if (units < 8 * kSms) {
        parts = ceil_div(8 * kSms, units);
        if (parts > ceil_div(blocks, 32)) parts = ceil_div(blocks, 32);
        parts = fewest_rounds(units, blocks, parts);
    }
    if (parts <= 1) return s;
    s.chunk = static_cast<int>(ceil_div(blocks, parts));
    s.parts = static_cast<int>(ceil_div(blocks, s.chunk));
    return s;
}

Split window_split(long long rows, long long n_seq, int heads, int kv_heads, int head_dim, long long max_slots, long long window,
                   long long sinks) {
    const int keys = keys_of(head_dim), tile = rows_of(head_dim);
    const long long group = heads / kv_heads;
    long long blocks = ceil_div(max_slots, keys);
    if (window > 0) {
        const long long some = ceil_div(window + ceil_div(tile, group), keys) + 1 + ceil_div(sinks, keys);
        if (some < blocks) blocks = some;
    }
    const long long tiles = n_seq > ceil_div(rows * group, tile) ? n_seq : ceil_div(rows * group, tile);
    const long long each = ceil_div(rows, n_seq) * group;
    return split(tiles * kv_heads, blocks, each < tile ? each : tile, keys);
}

struct PrefixSplit {
    Split own;
    int chunk, parts;
};

PrefixSplit prefix_split(long long n_seq, int heads, int kv_heads, int head_dim, long long max_slots, long long max_prefix) {
    const int keys = keys_of(head_dim), tile = rows_of(head_dim);
    const long long group = heads / kv_heads;
    PrefixSplit s{};
    s.own = split(n_seq * kv_heads * ceil_div(group, tile), ceil_div(max_slots, keys), group < tile ? group : tile, keys);
    if (s.own.parts == 0) s.own = Split{INT_MAX, 1};
    // a few units a CTA at most, and of no less than a few blocks
    const long long blocks = ceil_div(max_prefix, keys), tiles = kv_heads * ceil_div(n_seq * group, tile);
    const long long a = ceil_div(4 * kSms, tiles), b = ceil_div(blocks, 4);
    s.chunk = static_cast<int>(ceil_div(blocks, fewest_rounds(tiles, blocks, a < b ? a : b)));
    s.parts = static_cast<int>(ceil_div(blocks, s.chunk));
    return s;
}

// Single tokens of groups up to so many heads go to the kernel for them, which hides latencies with several small CTAs an SM
// (behind a window of 2048, 64 x 8 groups of 4 heads: 86 us there, 145 here); it reads a larger group's pages more than once.
constexpr int kTokenGroup = 16;

// Whether the sequences' own slots behind a prefix go to that kernel too: where they are units enough to fill the GPU, for which
// another launch pays (us here and there: 160 units of up to 400 slots 29 and 33, 320 of up to 30 33 and 28, 512 of up to 1024 85
// and 64).
bool own_by_tokens(long long n_seq, int heads, int kv_heads) { return heads / kv_heads <= kTokenGroup && n_seq * kv_heads >= 2 * kSms; }

size_t up16(size_t v) { return (v + 15) & ~size_t(15); }
size_t parts_bytes(size_t rows, size_t heads, size_t head_dim, size_t parts) {
    return up16(rows * heads * parts * 2 * sizeof(float)) + rows * heads * parts * head_dim * sizeof(float);
}
constexpr size_t kBrokenBytes = 16;   // of TileParams::broken, behind the parts

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

// Boxes of 64 dims x `heads` heads x `tokens` rows of q; 128-byte swizzle.
bool map_queries(CUtensorMap* m, const TileParams& p, int head_dim, uint32_t dtype, int heads, int tokens) {
    const fer::host::EncodeTiledFn fn = fer::host::encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(p.heads), static_cast<cuuint64_t>(p.rows)};
    const cuuint64_t strides[2] = {2ull * head_dim, 2ull * p.qs};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(tokens)}, step[3] = {1, 1, 1};
    return fn(m, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p.q), dims,
              strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t run(const Paged& c, TileParams& p, cudaStream_t s) {
    using C = Cut<D>;
    static std::atomic<bool> known[fer::host::kMaxDevices];
    cudaError_t e = fer::host::allow_smem(reinterpret_cast<const void*>(attn_tiles<T, D>), C::kSmem, known);
    if (e != cudaSuccess) return e;
    CUtensorMap k_map, v_map, q_map{}, q_few_map{};
    const int rows = C::kKeys < c.page_size() ? C::kKeys : c.page_size();
    const uint32_t dtype = __is_same(T, __half) ? 1 : 2;
    if (!map_pages(&k_map, c, c.k, dtype, rows) || !map_pages(&v_map, c, c.v, dtype, rows)) return cudaErrorInvalidValue;
    const bool aligned = (reinterpret_cast<uintptr_t>(p.q) | (p.qs * 2)) % 16 == 0 && p.qs * 2 < (1ull << 40);
    p.q_maps = !aligned ? kQLoads : 128 % p.group == 0 ? kQBoxes : kQRows;
    if (p.q_maps == kQBoxes) {
        // a group of 64 or 128 has no unit of few rows
        if (!map_queries(&q_map, p, D, dtype, p.group, 128 / p.group) ||
            !map_queries(&q_few_map, p, D, dtype, p.group < 32 ? p.group : 32, p.group < 32 ? 32 / p.group : 1))
            return cudaErrorInvalidValue;
    } else if (p.q_maps == kQRows && !map_queries(&q_map, p, D, dtype, 1, 1)) {
        return cudaErrorInvalidValue;
    }
    // no more CTAs than there can be units
    const long long tiles = ceil_div(static_cast<long long>(p.rows) * p.group, C::kRows) + p.n_seq;
    long long most = tiles * c.kv_heads * (p.parts > 0 ? p.parts : 1);
    const int grid = static_cast<int>(most < kSms ? most : kSms);
    e = fer::host::launch_pdl(attn_tiles<T, D>, dim3(grid), dim3(C::kThreads), C::kSmem, s, c, p, k_map, v_map, q_map, q_few_map);
    if (e == cudaSuccess && p.parts > 0) {
        const long long ctas = ceil_div(static_cast<long long>(p.rows) * p.heads, kJoinWarps);
        e = fer::host::launch_pdl(attn_join<T, D>, dim3(static_cast<unsigned>(ctas)), dim3(32 * kJoinWarps), 0, s, c, p,
                                  __is_same(T, __half) ? 8.0f : 0.0f);
    }
    return e;
}

template <typename T>
cudaError_t run_dim(const Paged& c, TileParams& p, cudaStream_t s) {
    switch (c.head_dim) {
        case 64: return run<T, 64>(c, p, s);
        case 128: return run<T, 128>(c, p, s);
        default: return run<T, 256>(c, p, s);
    }
}

Divide divide(uint32_t by) {
    Divide d{by, 0, 0};
    while ((1u << d.shift) < by) ++d.shift;
    d.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << d.shift) - by)) / by + 1);
    return d;
}

// What both operators' arguments have in common.
cudaError_t common(const fer_paged_view_t* cache, const void* q, void* out, size_t q_stride, size_t out_stride, int heads,
                   float scale, const float* lse, Paged* c, TileParams* p) {
    const cudaError_t e = fer::host::paged_params(cache, c);
    if (e != cudaSuccess) return e;
    if (!q || !out || heads <= 0 || heads % c->kv_heads || heads > 65536) return cudaErrorInvalidValue;
    const size_t width = static_cast<size_t>(heads) * c->head_dim;
    if (q_stride < width || out_stride < width || !(scale >= 0.0f) || scale > kMostScale) return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 2 || !fer::host::words_aligned({lse}))
        return cudaErrorInvalidValue;
    if (c->kv_heads > 65535) return cudaErrorNotSupported;
    p->q = q;
    p->out = out;
    p->qs = q_stride;
    p->os = out_stride;
    p->lse = const_cast<float*>(lse);
    p->heads = heads;
    p->group = heads / c->kv_heads;
    p->by_group = divide(static_cast<uint32_t>(p->group));
    p->own_chunk_log2 = -1;
    p->scale2 = (scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(c->head_dim)) : scale) * kLog2e;
    return cudaSuccess;
}

// Units are counted in 31 bits, and so are the joining's CTAs.
bool countable(const Paged& c, const TileParams& p) {
    const long long tiles = ceil_div(static_cast<long long>(p.rows) * p.group, rows_of(c.head_dim)) + p.n_seq;
    return tiles * c.kv_heads * (p.parts > 0 ? p.parts : 1) <= INT_MAX - 65536ll &&
           static_cast<long long>(p.rows) * p.group <= INT_MAX - 65536ll &&
           ceil_div(static_cast<long long>(p.rows) * p.heads, kJoinWarps) <= INT_MAX;
}

cudaError_t go(const Paged& c, TileParams& p, uint32_t dtype, void* workspace, size_t bytes, cudaStream_t s) {
    if (!countable(c, p)) return cudaErrorNotSupported;
    if (p.parts > 0) {
        const size_t all = parts_bytes(p.rows, p.heads, c.head_dim, p.parts);
        if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || bytes < all + (p.offsets ? kBrokenBytes : 0))
            return cudaErrorInvalidValue;
        if (p.offsets) p.broken = reinterpret_cast<int*>(static_cast<char*>(workspace) + all);
        p.part_ml = static_cast<float*>(workspace);
        p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                            up16(static_cast<size_t>(p.rows) * p.heads * p.parts * 2 * sizeof(float)));
    }
    return dtype == 1 ? run_dim<__half>(c, p, s) : run_dim<__nv_bfloat16>(c, p, s);
}

bool sizes_ok(int heads, int kv_heads, int head_dim) {
    return heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

}  // namespace

extern "C" size_t fer_paged_window_attention_workspace_bytes(int rows, int n_seq, int heads, int kv_heads, int head_dim,
                                                             int max_slots, int window, int sinks) {
    if (rows <= 0 || n_seq <= 0 || max_slots <= 0 || window < 0 || sinks < 0 || !sizes_ok(heads, kv_heads, head_dim)) return 0;
    const Split s = window_split(rows, n_seq, heads, kv_heads, head_dim, max_slots, window, sinks);
    size_t n = s.parts > 0 ? parts_bytes(rows, heads, head_dim, s.parts) + kBrokenBytes : 16;
    if (rows == n_seq && heads / kv_heads <= kTokenGroup) {   // there may be no offsets
        const size_t m = fer::host::window_token_bytes(n_seq, heads, head_dim, max_slots, window, sinks);
        if (m > n) n = m;
    }
    return n;
}

extern "C" cudaError_t fer_paged_window_attention(const fer_paged_view_t* cache, const fer_paged_window_args_t* a, uint32_t* err,
                                                  cudaStream_t s) {
    if (!a) return cudaErrorInvalidValue;
    Paged c{};
    TileParams p{};
    const cudaError_t e = common(cache, a->q, a->out, a->q_stride, a->out_stride, a->heads, a->scale, a->lse, &c, &p);
    if (e != cudaSuccess) return e;
    if (a->rows < 0 || a->n_seq < 0 || a->n_seq > cache->batch || a->window < 0 || a->sinks < 0 ||
        (!a->offsets && a->rows != a->n_seq) || !fer::host::words_aligned({a->offsets}))
        return cudaErrorInvalidValue;
    if (a->rows == 0 || a->n_seq == 0) return cudaSuccess;
    if (a->n_seq > 65535) return cudaErrorNotSupported;
    if (!a->offsets && p.group <= kTokenGroup) {
        const cudaError_t t = fer::host::window_token(c, cache->dtype, *a, err, s);
        if (t != cudaErrorNotSupported) return t;   // its units are counted by the table's width, here by what is seen
    }
    p.offsets = a->offsets;
    p.rows = a->rows;
    p.n_seq = a->n_seq;
    p.window = a->window > 0 ? a->window : INT_MAX;
    p.sinks = a->window > 0 ? a->sinks : 0;
    p.err = err;
    const Split sp = window_split(a->rows, a->n_seq, a->heads, c.kv_heads, c.head_dim, c.max_slots(), a->window, a->sinks);
    p.chunk = sp.chunk;
    p.parts = sp.parts;
    return go(c, p, cache->dtype, a->workspace, a->workspace_bytes, s);
}

extern "C" size_t fer_paged_prefix_attention_workspace_bytes(int n_seq, int heads, int kv_heads, int head_dim, int max_slots,
                                                             int max_prefix_slots) {
    if (n_seq <= 0 || max_slots <= 0 || max_prefix_slots <= 0 || !sizes_ok(heads, kv_heads, head_dim)) return 0;
    const PrefixSplit s = prefix_split(n_seq, heads, kv_heads, head_dim, max_slots, max_prefix_slots);
    if (own_by_tokens(n_seq, heads, kv_heads))
        return parts_bytes(n_seq, heads, head_dim, s.parts) + fer::host::window_token_bytes(n_seq, heads, head_dim, max_slots, 0, 0);
    return parts_bytes(n_seq, heads, head_dim, static_cast<size_t>(s.own.parts) + s.parts);
}

extern "C" cudaError_t fer_paged_prefix_attention(const fer_paged_view_t* cache, const fer_paged_prefix_args_t* a, uint32_t* err,
                                                  cudaStream_t s) {
    if (!a) return cudaErrorInvalidValue;
    Paged c{};
    TileParams p{};
    const cudaError_t e = common(cache, a->q, a->out, a->q_stride, a->out_stride, a->heads, a->scale, a->lse, &c, &p);
    if (e != cudaSuccess) return e;
    if (!a->prefix_pages || !a->prefix_length || a->max_prefix_pages <= 0 || a->n_seq < 0 || a->n_seq > cache->batch ||
        !fer::host::words_aligned({a->prefix_pages, a->prefix_length}))
        return cudaErrorInvalidValue;
    const long long most = static_cast<long long>(a->max_prefix_pages) << c.shift;
    if (most > INT_MAX - 65536ll || a->n_seq > 65535) return cudaErrorNotSupported;
    if (a->n_seq == 0) return cudaSuccess;
    p.rows = p.n_seq = a->n_seq;
    p.window = INT_MAX;
    p.err = err;
    p.prefix_pages = a->prefix_pages;
    p.prefix_length = a->prefix_length;
    p.prefix_max = a->max_prefix_pages;
    const PrefixSplit sp = prefix_split(a->n_seq, a->heads, c.kv_heads, c.head_dim, c.max_slots(), most);
    p.prefix_chunk = sp.chunk;
    if (own_by_tokens(a->n_seq, a->heads, c.kv_heads)) {
        const int max_slots = c.max_slots(), chunk = fer::host::token_parts_chunk(max_slots);
        p.chunk = INT_MAX;
        p.parts = sp.parts;
        if (!countable(c, p)) return cudaErrorNotSupported;
        const size_t mine = parts_bytes(a->n_seq, a->heads, c.head_dim, sp.parts);
        if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 ||
            a->workspace_bytes < mine + fer::host::window_token_bytes(a->n_seq, a->heads, c.head_dim, max_slots, 0, 0))
            return cudaErrorInvalidValue;
        char* const at = static_cast<char*>(a->workspace) + mine;
        p.own_parts = (max_slots - 1) / chunk + 1;
        p.own_chunk_log2 = 0;
        while ((1 << p.own_chunk_log2) < chunk) ++p.own_chunk_log2;
        p.own_ml = reinterpret_cast<const float*>(at);
        p.own_o = reinterpret_cast<const float*>(at + up16(static_cast<size_t>(a->n_seq) * a->heads * p.own_parts * 2 * sizeof(float)));
        fer_paged_window_args_t own{};
        own.q = a->q;
        own.out = a->out;
        own.q_stride = a->q_stride;
        own.out_stride = a->out_stride;
        own.rows = own.n_seq = a->n_seq;
        own.heads = a->heads;
        own.scale = a->scale;
        own.lse = a->lse;
        own.workspace = at;
        const cudaError_t t = fer::host::token_parts(c, cache->dtype, own, err, s);
        if (t != cudaSuccess) return t;
        return go(c, p, cache->dtype, a->workspace, mine, s);
    }
    p.chunk = sp.own.chunk;
    p.own_parts = sp.own.parts;
    p.parts = sp.own.parts + sp.parts;
    return go(c, p, cache->dtype, a->workspace, a->workspace_bytes, s);
}
