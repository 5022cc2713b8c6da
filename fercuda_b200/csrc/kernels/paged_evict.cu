// Eviction from a paged cache by accumulated attention weight.
//
// Every (sequence, key head) of n > budget slots keeps `budget` of them: a
// selection over n keys, then the move of the kept rows that lie behind the
// budget into the rows freed before it. Sources lie at or behind `budget` and
// targets before it, so all moves are independent. What has to be read is 8
// bytes a slot (weight, position), and 2 x 2 x head_dim elements a moved row.
//
// A slot's key is 32 bits: all ones for a recent one, else the weight's bits
// in an order of unsigned integers (NaN 0). The selection finds the budget-th
// largest key by four 8-bit digits, counting in shared memory, and how many of
// the slots of exactly that key are kept: the lowest ones.
#include "paged.cuh"
#include "pdl.cuh"

#include <cstdint>

namespace {

using fer::dev::Paged;
constexpr int kSelect = 1024;   // threads of the selection
constexpr int kMove = 256;

struct EvictParams {
    int budget, recent, cap;     // cap: moves a (sequence, key head) can have
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

// Exclusive prefix sum over the block of two 16-bit counts packed in one word
// (each total fits 16 bits), and the totals.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* sh, uint32_t* total) {
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    uint32_t x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[w] = x;
    __syncthreads();
    if (w == 0) {
        uint32_t y = sh[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t z = __shfl_up_sync(0xffffffffu, y, off);
            if (lane >= off) y += z;
        }
        sh[lane] = y;
    }
    __syncthreads();
    *total = sh[31];
    return x - v + (w ? sh[w - 1] : 0u);
}

// grid (kv_heads, batch)
__global__ void __launch_bounds__(kSelect) evict_select(const Paged c, const EvictParams p) {
    __shared__ int s_hist[256];
    __shared__ uint32_t s_scan[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left;
    const int t = threadIdx.x, b = blockIdx.y;
    const size_t bh = static_cast<size_t>(b) * c.kv_heads + blockIdx.x;
    fer::dev::pdl_begin();
    bool bad;
    const int n = c.length(b, &bad);
    if (bad && t == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    const size_t most = static_cast<size_t>(c.max_slots());
    const float* w = p.weights + bh * most;
    const int32_t* pos = p.positions + bh * most;
    float* nw = p.new_weights + bh * most;
    int32_t* np = p.new_positions + bh * most;
    if (n <= p.budget) {
        for (int j = t; j < n; j += kSelect) {
            if (nw != w) nw[j] = w[j];
            if (np != pos) np[j] = pos[j];
        }
        if (t == 0) p.counts[bh] = 0;
        return;
    }
    const long long first = static_cast<long long>(p.seen[b]) - p.recent;
    if (t == 0) s_prefix = 0u, s_left = p.budget;
    for (int d = 24; d >= 0; d -= 8) {
        if (t < 256) s_hist[t] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        const int left = s_left;
        for (int j = t; j < n; j += kSelect) {
            const uint32_t k = key_of(w[j], pos[j], first);
            if (d == 24 || (k >> (d + 8)) == (prefix >> (d + 8))) atomicAdd(&s_hist[(k >> d) & 255u], 1);
        }
        __syncthreads();
        if (t == 0) {
            int above = 0, digit = 255;
            while (digit > 0 && above + s_hist[digit] < left) above += s_hist[digit--];
            s_prefix = prefix | static_cast<uint32_t>(digit) << d;
            s_left = left - above;
        }
        __syncthreads();
    }
    const uint32_t cut = s_prefix;
    const int ties = s_left;   // slots of key `cut` that are kept, the lowest first
    int seen_ties = 0, freed = 0, moved = 0;
    int32_t* to = p.to + bh * p.cap;
    int32_t* from = p.from + bh * p.cap;
    for (int j0 = 0; j0 < n; j0 += kSelect) {
        const int j = j0 + t;
        const uint32_t k = j < n ? key_of(w[j], pos[j], first) : 0u;
        uint32_t total;
        const uint32_t before = block_scan(j < n && k == cut ? 1u : 0u, s_scan, &total);
        const bool kept = j < n && (k > cut || (k == cut && seen_ties + static_cast<int>(before) < ties));
        seen_ties += total;
        const bool front = j < p.budget;
        const bool hole = j < n && front && !kept, mover = kept && !front;
        const uint32_t at = block_scan((hole ? 1u : 0u) | (mover ? 0x10000u : 0u), s_scan, &total);
        const int nth_hole = freed + static_cast<int>(at & 0xffffu), nth_mover = moved + static_cast<int>(at >> 16);
        if (hole && nth_hole < p.cap) to[nth_hole] = j;
        if (mover && nth_mover < p.cap) from[nth_mover] = j;
        freed += total & 0xffffu;
        moved += total >> 16;
        if (kept && front) {
            if (nw != w) nw[j] = w[j];
            if (np != pos) np[j] = pos[j];
        }
    }
    if (t == 0) p.counts[bh] = min(moved, min(freed, p.cap));   // all equal, unless the arrays changed meanwhile
}

// grid (move tiles, kv_heads, batch): a warp a row
template <int D>
__global__ void __launch_bounds__(kMove) evict_move(const Paged c, const EvictParams p) {
    fer::dev::pdl_begin();
    const int b = blockIdx.z, h = blockIdx.y, t = threadIdx.x;
    const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
    const size_t most = static_cast<size_t>(c.max_slots());
    const int moved = p.counts[bh];
    if (h == 0 && blockIdx.x == 0 && t == 0) {
        bool bad;
        const int n = c.length(b, &bad);
        p.new_lengths[b] = n < p.budget ? n : p.budget;
    }
    for (int i = blockIdx.x * (kMove / 32) + (t >> 5); i < moved; i += gridDim.x * (kMove / 32)) {
        const int from = p.from[bh * p.cap + i], to = p.to[bh * p.cap + i];
        const int pf = c.page(b, from), pt = c.page(b, to);
        if ((t & 31) == 0) {
            p.new_weights[bh * most + to] = p.weights[bh * most + from];
            p.new_positions[bh * most + to] = p.positions[bh * most + from];
            if (pf < 0 || pt < 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
        }
        if (pf < 0 || pt < 0) continue;
        const size_t src = c.row(pf, h, from), dst = c.row(pt, h, to);
        for (int e = (t & 31) * 8; e < 2 * D; e += 256) {   // the row's key, then its value
            uint16_t* base = static_cast<uint16_t*>(e < D ? c.k : c.v);
            const int q = e < D ? e : e - D;
            *reinterpret_cast<uint4*>(base + dst + q) = *reinterpret_cast<const uint4*>(base + src + q);
        }
    }
}

int most_moves(int max_slots, int budget) {
    const int behind = max_slots - budget;
    return behind < budget ? behind : budget;
}

size_t up16(size_t v) { return (v + 15) & ~size_t(15); }

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
    const int max_slots = c.max_pages << c.shift;
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
    cudaError_t e = fer::host::launch_pdl(evict_select, dim3(c.kv_heads, cache->batch), dim3(kSelect), 0, s, c, p);
    if (e != cudaSuccess) return e;
    const int tiles = p.cap / 64 + 1;   // eight rows a warp
    const dim3 grid(tiles, c.kv_heads, cache->batch);
    switch (c.head_dim) {
        case 64: e = fer::host::launch_pdl(evict_move<64>, grid, dim3(kMove), 0, s, c, p); break;
        case 128: e = fer::host::launch_pdl(evict_move<128>, grid, dim3(kMove), 0, s, c, p); break;
        default: e = fer::host::launch_pdl(evict_move<256>, grid, dim3(kMove), 0, s, c, p); break;
    }
    return e != cudaSuccess ? e : cudaGetLastError();
}
