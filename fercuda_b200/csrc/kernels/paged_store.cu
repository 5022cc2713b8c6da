// Store of new keys and values into a paged cache.
//
// Row r of sequence b goes to slot lengths[b] + (r - offsets[b]) of every key
// head: each byte is read once and written once, so the store is bound by HBM
// for prompts and by launch latency for a decode step.
//
// A CTA takes a run of rows. One thread a row finds its sequence (binary
// search in the offsets), slot and page; then a warp takes a row (several
// warps where rows are few) and walks its 16-byte pieces, kAhead of keys and
// of values in flight a lane: reads are contiguous along a row and writes
// along a head's row in its page. Weights and positions are walked with the
// row innermost: consecutive slots of a head are consecutive. Short rows are
// walked as one run of pieces by the whole CTA.
//
// Lengths: a CTA of a step (one row a sequence) is the only reader of its
// sequences' lengths and writes the new ones itself, in place or not. With
// offsets a sequence may span CTAs; then the first CTA's threads write the
// new lengths when they go elsewhere, and a second small kernel when they
// replace the old (2 us more).
//
// Measured: 37 prompts of 1 to 2048 rows of 8 heads x 128 f16 52.6 to 54.4 us,
// 88 to 91% of the HBM copy rate; a step of 64 rows of 16 heads x 64 4.6 us, the
// host's time for the call.
#include "paged.cuh"
#include "pdl.cuh"

#include <cstdint>

namespace {

using fer::dev::Paged;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRows = 128;  // rows a CTA at most
constexpr int kAhead = 4;
constexpr int kShort = 32 * kAhead;   // pieces of a row below which a CTA's rows are walked as one

struct StoreParams {
    const uint16_t* k_rows;
    const uint16_t* v_rows;
    size_t ks, vs;
    int rows, n_seq, run;      // run: rows a CTA
    uint32_t inverse;          // ceil(2^32 / pieces of a row), for short ones
    const int32_t* offsets;
    int32_t* new_lengths;
    float* weights;
    int32_t* positions;
    const int32_t* seen;
    int32_t* new_seen;
    uint32_t* err;
};

// Rows of sequence b, with offsets that are not in order counted as none.
__device__ __forceinline__ int row_lo(const StoreParams& p, int b) {
    const int o = p.offsets[b];
    return o < 0 ? 0 : o > p.rows ? p.rows : o;
}
__device__ __forceinline__ int new_rows(const StoreParams& p, int b) {
    if (!p.offsets) return b < p.rows ? 1 : 0;
    const int n = row_lo(p, b + 1) - row_lo(p, b);
    return n < 0 ? 0 : n;
}

__device__ __forceinline__ void advance(const Paged& c, const StoreParams& p, int b) {
    bool off;
    const int n = new_rows(p, b), most = c.max_slots(), len = c.length(b, &off);
    if (off) fer::dev::report(p.err, fer::dev::kErrBadShape);   // of a sequence without new rows as well
    p.new_lengths[b] = n > most - len ? most : len + n;
    if (p.new_seen) p.new_seen[b] = p.seen[b] + n;
}

template <typename Piece>
__global__ void __launch_bounds__(kThreads) store_rows(const Paged c, const StoreParams p, const bool update) {
    constexpr int kPer = sizeof(Piece) / 2;
    __shared__ int s_seq[kMaxRows], s_slot[kMaxRows], s_page[kMaxRows], s_pos[kMaxRows];
    const int t = threadIdx.x;
    fer::dev::pdl_begin();
    const int r0 = blockIdx.x * p.run;
    const int nr = min(p.run, p.rows - r0);
    uint32_t bad = 0;
    if (t < nr) {
        const int r = r0 + t;
        int b = r, at = 0;
        if (p.offsets) {
            // the last sequence that starts at or before r
            int lo = 0, hi = p.n_seq;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (row_lo(p, mid) <= r) lo = mid + 1;
                else hi = mid;
            }
            b = lo - 1;
            at = b >= 0 ? r - row_lo(p, b) : 0;
            if (b >= 0 && at >= new_rows(p, b)) b = -1;   // behind the last sequence
        }
        int page = -1, slot = 0, pos = 0;
        if (b >= 0) {
            bool off;
            const int len = c.length(b, &off);
            if (off) bad = fer::dev::kErrBadShape;
            if (at >= c.max_slots() - len) {
                bad = fer::dev::kErrBadShape;
                b = -1;
            } else {
                slot = len + at;
                page = c.page(b, slot);
                if (page < 0) bad = fer::dev::kErrBadShape;
                if (p.positions) pos = p.seen[b] + at;
            }
        }
        s_seq[t] = b;
        s_slot[t] = slot;
        s_page[t] = page;
        s_pos[t] = pos;
    }
    if (bad) fer::dev::report(p.err, bad);
    __syncthreads();
    // head_dim is a power of two: piece q of a row is piece q % pieces of head q / pieces
    const int pieces = c.head_dim / kPer, log = 31 - __clz(pieces), per_row = c.kv_heads << log;
    const int lane = t & 31, w = t >> 5, share = max(1, kWarps / p.run);   // warps a row
    if (per_row < kShort) {
        // i / per_row: exact, as i * per_row < kMaxRows * kShort^2 < 2^32; one piece a row does not occur
        const size_t head = static_cast<size_t>(pieces) << c.shift;
        for (int i0 = t; i0 < nr * per_row; i0 += kThreads * kAhead) {
            Piece kk[kAhead], vv[kAhead];
            int j[kAhead], q[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + kThreads * k;
                j[k] = static_cast<int>(__umulhi(static_cast<uint32_t>(i), p.inverse));
                q[k] = i - j[k] * per_row;
                if (i >= nr * per_row || s_page[j[k]] < 0) {
                    j[k] = -1;
                    continue;
                }
                const size_t r = r0 + static_cast<size_t>(j[k]);
                kk[k] = reinterpret_cast<const Piece*>(p.k_rows + r * p.ks)[q[k]];
                vv[k] = reinterpret_cast<const Piece*>(p.v_rows + r * p.vs)[q[k]];
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (j[k] < 0) continue;
                const size_t at = c.row(s_page[j[k]], 0, s_slot[j[k]]) / kPer + (q[k] >> log) * head + (q[k] & (pieces - 1));
                static_cast<Piece*>(c.k)[at] = kk[k];
                static_cast<Piece*>(c.v)[at] = vv[k];
            }
        }
    } else {
        for (int j = w / share; j < nr; j += max(1, kWarps / share)) {
            if (s_page[j] < 0) continue;
            const Piece* const kr = reinterpret_cast<const Piece*>(p.k_rows + (r0 + static_cast<size_t>(j)) * p.ks);
            const Piece* const vr = reinterpret_cast<const Piece*>(p.v_rows + (r0 + static_cast<size_t>(j)) * p.vs);
            const size_t to = c.row(s_page[j], 0, s_slot[j]) / kPer, head = static_cast<size_t>(pieces) << c.shift;
            Piece* const kp = static_cast<Piece*>(c.k) + to;
            Piece* const vp = static_cast<Piece*>(c.v) + to;
            for (int q0 = (w % share) * 32 + lane; q0 < per_row; q0 += 32 * share * kAhead) {
                Piece kk[kAhead], vv[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int q = q0 + 32 * share * k;
                    if (q < per_row) kk[k] = kr[q], vv[k] = vr[q];
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int q = q0 + 32 * share * k;
                    if (q >= per_row) break;
                    const size_t at = (q >> log) * head + (q & (pieces - 1));
                    kp[at] = kk[k];
                    vp[at] = vv[k];
                }
            }
        }
    }
    if (p.weights || p.positions) {
        const size_t most = static_cast<size_t>(c.max_slots());
        for (int i = t; i < nr * c.kv_heads; i += kThreads) {
            const int h = i / nr, j = i - h * nr;
            if (s_seq[j] < 0) continue;
            const size_t at = (static_cast<size_t>(s_seq[j]) * c.kv_heads + h) * most + s_slot[j];
            if (p.weights) p.weights[at] = 0.0f;
            if (p.positions) p.positions[at] = s_pos[j];
        }
    }
    if (!update) return;
    if (p.offsets) {
        // n_seq sequences over all CTAs; nothing in this launch reads what is written
        for (int b = blockIdx.x * kThreads + t; b < p.n_seq; b += gridDim.x * kThreads) advance(c, p, b);
    } else {
        // this CTA's own sequences; their lengths were read before the barrier
        if (t < nr) advance(c, p, r0 + t);
    }
}

__global__ void __launch_bounds__(kThreads) advance_lengths(const Paged c, const StoreParams p) {
    fer::dev::pdl_begin();
    const int b = blockIdx.x * kThreads + threadIdx.x;
    if (b < p.n_seq) advance(c, p, b);
}

}  // namespace

extern "C" cudaError_t fer_paged_store(const fer_paged_view_t* cache, const fer_paged_store_args_t* a, uint32_t* err,
                                       cudaStream_t s) {
    Paged c{};
    const cudaError_t ce = fer::host::paged_params(cache, &c);
    if (ce != cudaSuccess) return ce;
    if (!a || a->rows < 0 || a->n_seq < 0 || a->n_seq > cache->batch || !a->new_lengths) return cudaErrorInvalidValue;
    if (!a->offsets && a->rows != a->n_seq) return cudaErrorInvalidValue;
    if (a->positions && (!a->seen || !a->new_seen)) return cudaErrorInvalidValue;
    if (!fer::host::words_aligned({a->offsets, a->new_lengths, a->weights, a->positions, a->seen, a->new_seen}))
        return cudaErrorInvalidValue;
    const size_t width = static_cast<size_t>(c.kv_heads) * c.head_dim;
    if (a->rows > 0 && (!a->k_rows || !a->v_rows || a->k_stride < width || a->v_stride < width))
        return cudaErrorInvalidValue;
    if (a->n_seq == 0) return cudaSuccess;
    if (c.kv_heads > (1 << 16)) return cudaErrorNotSupported;
    const uintptr_t rows_at = reinterpret_cast<uintptr_t>(a->k_rows) | reinterpret_cast<uintptr_t>(a->v_rows);
    if (rows_at % 2) return cudaErrorInvalidValue;
    StoreParams p{};
    p.k_rows = static_cast<const uint16_t*>(a->k_rows);
    p.v_rows = static_cast<const uint16_t*>(a->v_rows);
    p.ks = a->k_stride;
    p.vs = a->v_stride;
    p.rows = a->rows;
    p.n_seq = a->n_seq;
    p.offsets = a->offsets;
    p.new_lengths = a->new_lengths;
    p.weights = a->weights;
    p.positions = a->positions;
    p.seen = a->seen;
    p.new_seen = a->positions || a->seen ? a->new_seen : nullptr;
    p.err = err;
    const bool wide = rows_at % 16 == 0 && a->k_stride % 8 == 0 && a->v_stride % 8 == 0;
    const size_t per_row = wide ? width / 8 : width;
    p.inverse = static_cast<uint32_t>(((1ull << 32) + per_row - 1) / per_row);
    // 16 rows a CTA, more of short ones (of 8 pieces: 69.6 us for 131072 rows with 16, 20.5 with 128); fewer (and more
    // warps a row) where that would leave SMs without work
    p.run = 16;
    while (p.run < kMaxRows && p.run * per_row < 1024) p.run *= 2;
    while (p.run > 1 && a->rows < 148 * 2 * p.run) p.run /= 2;
    const bool in_place = a->new_lengths == cache->lengths || (p.new_seen && p.new_seen == a->seen);
    const bool later = a->offsets && in_place;
    cudaError_t e = cudaSuccess;
    if (a->rows > 0 || !later) {
        const int grid = a->rows > 0 ? (a->rows - 1) / p.run + 1 : 1;
        e = wide ? fer::host::launch_pdl(store_rows<uint4>, dim3(grid), dim3(kThreads), 0, s, c, p, !later)
                 : fer::host::launch_pdl(store_rows<uint16_t>, dim3(grid), dim3(kThreads), 0, s, c, p, !later);
        if (e != cudaSuccess) return e;
    }
    if (later)
        e = fer::host::launch_pdl(advance_lengths, dim3((a->n_seq + kThreads - 1) / kThreads), dim3(kThreads), 0, s, c, p);
    return e;
}
