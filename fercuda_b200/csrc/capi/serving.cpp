// Serving operators of a paged key-value cache: fer_submit_rotary,
// fer_submit_paged_store, fer_submit_paged_attention, fer_submit_paged_evict.
//
// Unknown ids -> NOT_FOUND; wrong dtypes, ranks, shapes, columns and
// overlapping outputs -> INVALID_ARGUMENT. Nothing is launched after a
// refusal.
#include "session.hpp"

#include "fercuda/b200/native.h"

#include <cfloat>
#include <climits>
#include <new>

using fer::capi::Buffer;
using fer::capi::Session;
using fer::capi::internal;
using fer::capi::invalid;
using fer::capi::not_found;
using fer::capi::ok;

namespace {

// Makes the session's device current for a call and restores the caller's.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
        if (before_ != device) cudaSetDevice(device);
        switched_ = before_ != device;
    }
    ~OnDevice() {
        if (switched_) cudaSetDevice(before_);
    }

  private:
    int before_ = 0;
    bool switched_ = false;
};

bool overlap(const Buffer* a, const Buffer* b) {
    const auto x = reinterpret_cast<uintptr_t>(a->ptr), y = reinterpret_cast<uintptr_t>(b->ptr);
    return x < y + b->bytes && y < x + a->bytes;
}

bool same(const Buffer* a, const Buffer* b) { return a->ptr == b->ptr && a->bytes == b->bytes; }

// A rank-2 buffer's columns [col, col + n).
struct Cols {
    const Buffer* buf = nullptr;
    uint64_t col = 0, n = 0;
    bool fits() const { return col + n <= buf->desc.dims[1]; }
    void* at() const {
        return static_cast<char*>(buf->ptr) + col * (buf->bytes / buf->numel);
    }
};

// Whether two column ranges share an element (judged by the whole buffers
// unless they are the same memory of the same width).
bool overlap(const Cols& a, const Cols& b) {
    if (!overlap(a.buf, b.buf)) return false;
    if (a.buf->ptr == b.buf->ptr && a.buf->desc.dims[1] == b.buf->desc.dims[1])
        return a.col < b.col + b.n && b.col < a.col + a.n;
    return true;
}

bool half_dtype(uint32_t dt) { return dt == FER_DTYPE_F16 || dt == FER_DTYPE_BF16; }

bool is_vector(const Buffer* b, uint32_t dtype, uint64_t n) {
    return b->desc.dtype == dtype && b->desc.rank == 1 && b->desc.dims[0] == n;
}

struct Cache {
    const Buffer *k = nullptr, *v = nullptr, *table = nullptr, *lengths = nullptr;
    fer_paged_view_t view{};
    uint64_t max_slots = 0;
    bool is_slots(const Buffer* b, uint32_t dtype) const {
        return b->desc.dtype == dtype && b->desc.rank == 3 && b->desc.dims[0] == static_cast<uint32_t>(view.batch) &&
               b->desc.dims[1] == static_cast<uint32_t>(view.kv_heads) && b->desc.dims[2] == max_slots;
    }
    bool touches(const Buffer* b) const {
        return overlap(b, k) || overlap(b, v) || overlap(b, table) || overlap(b, lengths);
    }
};

fer_status_t open_cache(const Session& S, const fer_paged_cache_t& r, Cache* c) {
    c->k = S.find(r.k);
    c->v = S.find(r.v);
    c->table = S.find(r.page_table);
    c->lengths = S.find(r.lengths);
    if (!c->k || !c->v || !c->table || !c->lengths) return not_found("buffer id not found");
    const fer_buffer_desc_t &k = c->k->desc, &v = c->v->desc, &t = c->table->desc;
    if (!half_dtype(k.dtype) || v.dtype != k.dtype) return invalid("paged cache requires f16 or bf16 keys and values");
    if (k.rank != 4 || v.rank != 4) return invalid("paged cache requires rank-4 keys and values");
    for (int i = 0; i < 4; ++i)
        if (k.dims[i] != v.dims[i]) return invalid("paged cache keys and values must have one shape");
    if (t.dtype != FER_DTYPE_I32 || t.rank != 2) return invalid("paged cache requires an i32 rank-2 page table");
    if (!is_vector(c->lengths, FER_DTYPE_I32, t.dims[0])) return invalid("paged cache requires i32 lengths [batch]");
    if (k.dims[3] != 64 && k.dims[3] != 128 && k.dims[3] != 256)
        return invalid("paged cache head_dim must be 64, 128 or 256");
    if (k.dims[2] < 8 || k.dims[2] > 256 || (k.dims[2] & (k.dims[2] - 1)))
        return invalid("paged cache page_size must be a power of two from 8 to 256");
    if (k.dims[0] > INT_MAX || k.dims[1] > 65535 || t.dims[0] > 65535 ||
        static_cast<uint64_t>(t.dims[1]) * k.dims[2] > INT_MAX - 65536)
        return invalid("paged cache is too large");
    if ((reinterpret_cast<uintptr_t>(c->k->ptr) | reinterpret_cast<uintptr_t>(c->v->ptr)) % 16)
        return invalid("paged cache keys and values must be 16-byte aligned");
    if (overlap(c->k, c->v) || overlap(c->k, c->table) || overlap(c->v, c->table) || overlap(c->k, c->lengths) ||
        overlap(c->v, c->lengths) || overlap(c->table, c->lengths))
        return invalid("paged cache buffers overlap");
    c->max_slots = static_cast<uint64_t>(t.dims[1]) * k.dims[2];
    fer_paged_view_t& w = c->view;
    w.k = c->k->ptr;
    w.v = c->v->ptr;
    w.page_table = static_cast<const int32_t*>(c->table->ptr);
    w.lengths = static_cast<const int32_t*>(c->lengths->ptr);
    w.batch = static_cast<int>(t.dims[0]);
    w.max_pages = static_cast<int>(t.dims[1]);
    w.pages = static_cast<int>(k.dims[0]);
    w.kv_heads = static_cast<int>(k.dims[1]);
    w.page_size = static_cast<int>(k.dims[2]);
    w.head_dim = static_cast<int>(k.dims[3]);
    w.dtype = k.dtype;
    return ok();
}

// An optional buffer: 0 gives null.
bool find_optional(const Session& S, uint64_t id, const Buffer** out) {
    *out = nullptr;
    if (!id) return true;
    *out = S.find(id);
    return *out != nullptr;
}

fer_status_t finish(Session& S, cudaError_t e, uint64_t* out_job_id) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        if (e == cudaErrorInvalidValue || e == cudaErrorNotSupported) return invalid("operator does not take this request");
        return internal("kernel launch failed");
    }
    uint64_t job = 0;
    const fer_status_t st = S.make_job({}, &job);
    if (st.code == FER_STATUS_OK && out_job_id) *out_job_id = job;
    return st;
}

// A job's completion event cannot be queried once it was captured.
bool capturing(const Session& S) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(S.stream, &st) != cudaSuccess) {
        cudaGetLastError();
        return true;
    }
    return st != cudaStreamCaptureStatusNone;
}

const char* const kCapturing = "session stream is being captured; use the launchers of native.h";

fer_status_t submit_rotary(Session& S, const fer_rotary_request_t& r, uint64_t* out_job_id) {
    const Buffer* x = S.find(r.x);
    const Buffer* o = S.find(r.out);
    const Buffer* pos = S.find(r.positions);
    if (!x || !o || !pos) return not_found("buffer id not found");
    if (x->desc.dtype != FER_DTYPE_F32 && !half_dtype(x->desc.dtype)) return invalid("rotary requires f32, f16 or bf16 buffers");
    if (o->desc.dtype != x->desc.dtype) return invalid("rotary requires matching dtypes for x/out");
    if (x->desc.rank != 2 || o->desc.rank != 2 || o->desc.dims[0] != x->desc.dims[0])
        return invalid("rotary requires rank-2 x and out of the same rows");
    if (x->desc.dims[0] > INT_MAX) return invalid("rotary takes at most 2^31 - 1 rows");
    if (r.axes < 1 || r.axes > 4) return invalid("rotary takes 1 to 4 axes");
    if (pos->desc.dtype != FER_DTYPE_I32 || pos->desc.dims[0] != x->desc.dims[0] ||
        !((pos->desc.rank == 1 && r.axes == 1) || (pos->desc.rank == 2 && pos->desc.dims[1] == r.axes)))
        return invalid("rotary requires i32 positions [rows, axes]");
    if (r.heads == 0 || r.heads > 65536 || r.head_dim == 0 || r.head_dim % 2 || r.head_dim > 1024)
        return invalid("rotary requires 1 to 65536 heads of an even head_dim of at most 1024");
    const uint32_t rot = r.rotary_dim ? r.rotary_dim : r.head_dim;
    if (rot % 2 || rot > r.head_dim) return invalid("rotary_dim must be even and at most head_dim");
    if (r.flags & ~(FER_ROTARY_INTERLEAVED | FER_ROTARY_AXIS_FREQS | FER_ROTARY_INVERSE))
        return invalid("unknown rotary flags");
    if (!(r.base > 0.0f) || r.base > FLT_MAX) return invalid("rotary base must be positive and finite");
    uint64_t sum = 0;
    for (uint32_t i = 0; i < r.axes; ++i) sum += r.sections[i];
    const bool whole = r.axes == 1 && r.sections[0] == 0;
    if (!whole && sum != rot / 2) return invalid("rotary sections must add up to rotary_dim / 2");
    const uint64_t width = static_cast<uint64_t>(r.heads) * r.head_dim;
    const Cols cx{x, r.x_col, width}, co{o, r.out_col, width};
    if (!cx.fits() || !co.fits()) return invalid("rotary heads reach past the columns");
    const bool in_place = x->ptr == o->ptr && x->desc.dims[1] == o->desc.dims[1] && r.x_col == r.out_col;
    if (!in_place && overlap(cx, co)) return invalid("rotary x and out overlap");
    if (overlap(o, pos)) return invalid("rotary out and positions overlap");
    fer_rotary_args_t a{};
    a.x = cx.at();
    a.out = co.at();
    a.positions = static_cast<const int32_t*>(pos->ptr);
    a.x_stride = x->desc.dims[1];
    a.out_stride = o->desc.dims[1];
    a.rows = static_cast<int>(x->desc.dims[0]);
    a.heads = static_cast<int>(r.heads);
    a.head_dim = static_cast<int>(r.head_dim);
    a.rotary_dim = static_cast<int>(rot);
    a.axes = static_cast<int>(r.axes);
    for (uint32_t i = 0; i < r.axes; ++i) a.sections[i] = static_cast<int>(whole ? rot / 2 : r.sections[i]);
    a.base = r.base;
    a.flags = r.flags;
    a.dtype = x->desc.dtype;
    if (capturing(S)) return invalid(kCapturing);
    return finish(S, fer_rotary(&a, S.stream), out_job_id);
}

fer_status_t submit_store(Session& S, const fer_paged_store_request_t& r, uint64_t* out_job_id) {
    Cache c;
    const fer_status_t st = open_cache(S, r.cache, &c);
    if (st.code != FER_STATUS_OK) return st;
    const Buffer* k = S.find(r.k_rows);
    const Buffer* v = S.find(r.v_rows);
    const Buffer *off, *len, *w, *pos, *seen, *nseen;
    if (!k || !v || !find_optional(S, r.offsets, &off) || !find_optional(S, r.new_lengths, &len) ||
        !find_optional(S, r.weights, &w) || !find_optional(S, r.positions, &pos) || !find_optional(S, r.seen, &seen) ||
        !find_optional(S, r.new_seen, &nseen))
        return not_found("buffer id not found");
    if (k->desc.dtype != c.view.dtype || v->desc.dtype != c.view.dtype)
        return invalid("paged store requires rows of the cache's dtype");
    if (k->desc.rank != 2 || v->desc.rank != 2 || k->desc.dims[0] != v->desc.dims[0] || k->desc.dims[0] > INT_MAX)
        return invalid("paged store requires rank-2 key and value rows of the same count");
    const uint64_t rows = k->desc.dims[0], width = static_cast<uint64_t>(c.view.kv_heads) * c.view.head_dim;
    const Cols ck{k, r.k_col, width}, cv{v, r.v_col, width};
    if (!ck.fits() || !cv.fits()) return invalid("paged store heads reach past the columns");
    uint64_t n_seq = rows;
    if (off) {
        if (off->desc.dtype != FER_DTYPE_I32 || off->desc.rank != 1 || off->desc.dims[0] < 2)
            return invalid("paged store requires i32 offsets [sequences + 1]");
        n_seq = off->desc.dims[0] - 1;
    }
    if (n_seq > static_cast<uint64_t>(c.view.batch)) return invalid("paged store has more sequences than the cache");
    if (!len) len = c.lengths;
    if (!is_vector(len, FER_DTYPE_I32, c.view.batch)) return invalid("paged store requires i32 new_lengths [batch]");
    if (w && !c.is_slots(w, FER_DTYPE_F32)) return invalid("paged weights must be f32 [batch, kv_heads, slots]");
    if (pos && !c.is_slots(pos, FER_DTYPE_I32)) return invalid("paged positions must be i32 [batch, kv_heads, slots]");
    if (pos && !seen) return invalid("paged positions require seen");
    if (seen && !nseen) nseen = seen;
    if (nseen && !seen) return invalid("paged new_seen requires seen");
    if (seen && (!is_vector(seen, FER_DTYPE_I32, c.view.batch) || !is_vector(nseen, FER_DTYPE_I32, c.view.batch)))
        return invalid("paged seen must be i32 [batch]");
    // what is written against everything else
    const Buffer* out[] = {c.k, c.v, len, w, pos, nseen};
    const Buffer* in[] = {c.table, c.lengths, k, v, off, seen};
    for (int i = 0; i < 6; ++i) {
        if (!out[i]) continue;
        for (int j = 0; j < i; ++j)
            if (out[j] && overlap(out[i], out[j])) return invalid("paged store buffers overlap");
        for (const Buffer* b : in) {
            if (!b || !overlap(out[i], b)) continue;
            if ((i == 2 && b == c.lengths && same(len, b)) || (i == 5 && b == seen && same(nseen, b))) continue;
            return invalid("paged store buffers overlap");
        }
    }
    fer_paged_store_args_t a{};
    a.k_rows = ck.at();
    a.v_rows = cv.at();
    a.k_stride = k->desc.dims[1];
    a.v_stride = v->desc.dims[1];
    a.rows = static_cast<int>(rows);
    a.n_seq = static_cast<int>(n_seq);
    a.offsets = off ? static_cast<const int32_t*>(off->ptr) : nullptr;
    a.new_lengths = static_cast<int32_t*>(len->ptr);
    a.weights = w ? static_cast<float*>(w->ptr) : nullptr;
    a.positions = pos ? static_cast<int32_t*>(pos->ptr) : nullptr;
    a.seen = seen ? static_cast<const int32_t*>(seen->ptr) : nullptr;
    a.new_seen = nseen ? static_cast<int32_t*>(nseen->ptr) : nullptr;
    if (capturing(S)) return invalid(kCapturing);
    return finish(S, fer_paged_store(&c.view, &a, S.dev_err, S.stream), out_job_id);
}

fer_status_t submit_attention(Session& S, const fer_paged_attention_request_t& r, uint64_t* out_job_id) {
    Cache c;
    const fer_status_t st = open_cache(S, r.cache, &c);
    if (st.code != FER_STATUS_OK) return st;
    const Buffer* q = S.find(r.q);
    const Buffer* o = S.find(r.out);
    const Buffer* ws = S.find(r.workspace);
    const Buffer *lse, *w;
    if (!q || !o || !ws || !find_optional(S, r.lse, &lse) || !find_optional(S, r.weights, &w))
        return not_found("buffer id not found");
    if (q->desc.dtype != c.view.dtype || o->desc.dtype != c.view.dtype)
        return invalid("paged attention requires q and out of the cache's dtype");
    if (q->desc.rank != 2 || o->desc.rank != 2 || q->desc.dims[0] != o->desc.dims[0])
        return invalid("paged attention requires rank-2 q and out of the same rows");
    const uint64_t rows = q->desc.dims[0];
    if (rows > static_cast<uint64_t>(c.view.batch)) return invalid("paged attention has more rows than the cache");
    if (r.heads == 0 || r.heads % static_cast<uint32_t>(c.view.kv_heads) || r.heads > 65536)
        return invalid("paged attention heads must be a multiple of kv_heads, at most 65536");
    if (!(r.scale >= 0.0f) || r.scale > 2.0e38f) return invalid("paged attention scale must be from 0 to 2e38");
    const uint64_t width = static_cast<uint64_t>(r.heads) * c.view.head_dim;
    const Cols cq{q, r.q_col, width}, co{o, r.out_col, width};
    if (!cq.fits() || !co.fits()) return invalid("paged attention heads reach past the columns");
    if (lse && !(lse->desc.dtype == FER_DTYPE_F32 && lse->desc.rank == 2 && lse->desc.dims[0] == rows &&
                 lse->desc.dims[1] == r.heads))
        return invalid("paged attention lse must be f32 [rows, heads]");
    if (w && !c.is_slots(w, FER_DTYPE_F32)) return invalid("paged weights must be f32 [batch, kv_heads, slots]");
    if (ws->desc.dtype != FER_DTYPE_U8) return invalid("workspace must be a u8 buffer");
    const uint64_t need = fer_paged_attention_workspace_bytes(static_cast<int>(rows), static_cast<int>(r.heads),
                                                              c.view.kv_heads, c.view.head_dim,
                                                              static_cast<int>(c.max_slots), w != nullptr);
    if (ws->bytes < need || reinterpret_cast<uintptr_t>(ws->ptr) % 16)
        return invalid("workspace is too small or not 16-byte aligned");
    if (overlap(cq, co)) return invalid("paged attention q and out overlap");
    const Buffer* out[] = {o, lse, w, ws};
    for (int i = 0; i < 4; ++i) {
        if (!out[i]) continue;
        if (c.touches(out[i]) || (i > 0 && overlap(out[i], q))) return invalid("paged attention buffers overlap");
        for (int j = 0; j < i; ++j)
            if (out[j] && overlap(out[i], out[j])) return invalid("paged attention buffers overlap");
    }
    fer_paged_attention_args_t a{};
    a.q = cq.at();
    a.out = co.at();
    a.q_stride = q->desc.dims[1];
    a.out_stride = o->desc.dims[1];
    a.n_seq = static_cast<int>(rows);
    a.heads = static_cast<int>(r.heads);
    a.scale = r.scale;
    a.lse = lse ? static_cast<float*>(lse->ptr) : nullptr;
    a.weights = w ? static_cast<float*>(w->ptr) : nullptr;
    a.workspace = ws->ptr;
    a.workspace_bytes = ws->bytes;
    if (capturing(S)) return invalid(kCapturing);
    return finish(S, fer_paged_attention(&c.view, &a, S.dev_err, S.stream), out_job_id);
}

fer_status_t submit_evict(Session& S, const fer_paged_evict_request_t& r, uint64_t* out_job_id) {
    Cache c;
    const fer_status_t st = open_cache(S, r.cache, &c);
    if (st.code != FER_STATUS_OK) return st;
    const Buffer* w = S.find(r.weights);
    const Buffer* pos = S.find(r.positions);
    const Buffer* seen = S.find(r.seen);
    const Buffer* ws = S.find(r.workspace);
    const Buffer *len, *nw, *np;
    if (!w || !pos || !seen || !ws || !find_optional(S, r.new_lengths, &len) || !find_optional(S, r.new_weights, &nw) ||
        !find_optional(S, r.new_positions, &np))
        return not_found("buffer id not found");
    if (!len) len = c.lengths;
    if (!nw) nw = w;
    if (!np) np = pos;
    if (!c.is_slots(w, FER_DTYPE_F32) || !c.is_slots(nw, FER_DTYPE_F32))
        return invalid("paged weights must be f32 [batch, kv_heads, slots]");
    if (!c.is_slots(pos, FER_DTYPE_I32) || !c.is_slots(np, FER_DTYPE_I32))
        return invalid("paged positions must be i32 [batch, kv_heads, slots]");
    if (!is_vector(seen, FER_DTYPE_I32, c.view.batch)) return invalid("paged seen must be i32 [batch]");
    if (!is_vector(len, FER_DTYPE_I32, c.view.batch)) return invalid("paged evict requires i32 new_lengths [batch]");
    if (r.budget < 1 || r.budget > INT_MAX || r.recent > r.budget)
        return invalid("paged evict requires 1 <= budget and recent <= budget");
    if (ws->desc.dtype != FER_DTYPE_U8) return invalid("workspace must be a u8 buffer");
    const uint64_t need = fer_paged_evict_workspace_bytes(c.view.batch, c.view.kv_heads, static_cast<int>(c.max_slots),
                                                          static_cast<int>(r.budget));
    if (ws->bytes < need || reinterpret_cast<uintptr_t>(ws->ptr) % 16)
        return invalid("workspace is too small or not 16-byte aligned");
    const Buffer* out[] = {c.k, c.v, len, nw, np, ws};
    const Buffer* in[] = {c.table, c.lengths, w, pos, seen};
    for (int i = 0; i < 6; ++i) {
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return invalid("paged evict buffers overlap");
        for (const Buffer* b : in) {
            if (!overlap(out[i], b)) continue;
            if ((i == 2 && b == c.lengths && same(len, b)) || (i == 3 && b == w && same(nw, b)) ||
                (i == 4 && b == pos && same(np, b)))
                continue;
            return invalid("paged evict buffers overlap");
        }
    }
    fer_paged_evict_args_t a{};
    a.budget = static_cast<int>(r.budget);
    a.recent = static_cast<int>(r.recent);
    a.weights = static_cast<const float*>(w->ptr);
    a.positions = static_cast<const int32_t*>(pos->ptr);
    a.seen = static_cast<const int32_t*>(seen->ptr);
    a.new_lengths = static_cast<int32_t*>(len->ptr);
    a.new_weights = static_cast<float*>(nw->ptr);
    a.new_positions = static_cast<int32_t*>(np->ptr);
    a.workspace = ws->ptr;
    a.workspace_bytes = ws->bytes;
    if (capturing(S)) return invalid(kCapturing);
    return finish(S, fer_paged_evict(&c.view, &a, S.dev_err, S.stream), out_job_id);
}

// The common frame of the entry points: null checks, the session's device,
// and no C++ exception past the C boundary.
template <typename Req, typename Fn>
fer_status_t entry(fer_session_t* session, const Req* req, uint64_t* out_job_id, Fn fn) {
    if (!session) return invalid("session is null");
    if (!req) return invalid("request is null");
    try {
        const OnDevice on(session->impl.device);
        return fn(session->impl, *req, out_job_id);
    } catch (const std::bad_alloc&) {
        return internal("allocation failure");
    } catch (...) {
        return internal("submit failure");
    }
}

}  // namespace

extern "C" {

fer_status_t fer_submit_rotary(fer_session_t* session, const fer_rotary_request_t* req, uint64_t* out_job_id) {
    return entry(session, req, out_job_id, submit_rotary);
}

fer_status_t fer_submit_paged_store(fer_session_t* session, const fer_paged_store_request_t* req,
                                    uint64_t* out_job_id) {
    return entry(session, req, out_job_id, submit_store);
}

fer_status_t fer_submit_paged_attention(fer_session_t* session, const fer_paged_attention_request_t* req,
                                        uint64_t* out_job_id) {
    return entry(session, req, out_job_id, submit_attention);
}

fer_status_t fer_submit_paged_evict(fer_session_t* session, const fer_paged_evict_request_t* req,
                                    uint64_t* out_job_id) {
    return entry(session, req, out_job_id, submit_evict);
}

}  // extern "C"
