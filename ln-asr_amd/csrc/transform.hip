// Feature transforms: entry points.  Checks, staging of host arrays and the sequence of products; the kernels are in
// transform_rows.hip and transform_grad.hip.
#include <algorithm>
#include <exception>

#include "transform.h"

namespace lnasr {

static_assert(sizeof(lnasr_ctx::tr_ws) / sizeof(DevBuf) == kTrCount, "workspaces of the feature transforms");

int transform_ws(lnasr_ctx* ctx, int i, size_t bytes, void** out) {
    DevBuf& b = ctx->tr_ws[i];
    if (bytes > b.cap || !b.p) {
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        LN_HIP(hipStreamIsCapturing(ctx->stream, &st));
        LN_REQUIRE(st == hipStreamCaptureStatusNone,
                   "a workspace of %zu bytes cannot be allocated while the stream is captured: run the call once before", bytes);
        if (ctx->tr_captured) {                           // (left to the graphs; twice as large, so that few are)
            bytes = std::max(bytes, 2 * b.cap);
            b = DevBuf();
        }
        LN_TRY(b.reserve(bytes));
    }
    *out = b.p;
    return 0;
}

namespace {

struct Call {
    lnasr_ctx* const ctx;
    bool capturing = false;
    struct Range { const char *lo, *hi; bool out; const char* what; };
    Range ranges[16];
    int n = 0;
    struct Back { void* host; void* dev; size_t bytes; };
    Back back[5];
    int nback = 0;
    bool pinned = false;                                  // a copy from pinned host memory is on its way
    std::unique_lock<std::mutex> lock;
    const bool prof;

    explicit Call(lnasr_ctx* c) : ctx(c), lock(c->tr_mutex), prof(c->prof_on) {}
    ~Call() {
        if (capturing) ctx->prof_on = prof;
    }

    int begin() {
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(ctx->stream, &st) != hipSuccess) {
            (void)hipGetLastError();
            return fail(LNASR_E_INVALID, "the default stream takes no calls while another stream is captured");
        }
        capturing = st != hipStreamCaptureStatusNone;
        if (capturing) {
            ctx->tr_captured = true;
            ctx->prof_on = false;                         // (its events would belong to the graph)
        }
        return 0;
    }
    // 1: memory of the context's device, 0: host memory, negative: error
    int place(const void* p, const char* what) {
        hipPointerAttribute_t at;
        if (hipPointerGetAttributes(&at, p) != hipSuccess) {
            (void)hipGetLastError();
            return 0;
        }
        if (at.type == hipMemoryTypeHost) pinned = true;
        if (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged) return 0;
        if (at.device != ctx->device)
            return fail(LNASR_E_INVALID, "%s lies on device %d, the context on device %d", what, at.device, ctx->device);
        return 1;
    }
    // No output may share memory with an input or another output: results are written while inputs are still read
    int note(const void* p, size_t bytes, bool out, const char* what) {
        const char *lo = (const char*)p, *hi = lo + bytes;
        for (int i = 0; i < n; ++i)
            if ((out || ranges[i].out) && lo < ranges[i].hi && ranges[i].lo < hi)
                return fail(LNASR_E_INVALID, "%s shares memory with %s", what, ranges[i].what);
        ranges[n++] = {lo, hi, out, what};
        return 0;
    }
    int in(const void* p, size_t bytes, int ws, const char* what, const void** out) {
        *out = nullptr;
        if (bytes == 0) return 0;
        LN_REQUIRE(p, "%s is null", what);
        LN_TRY(note(p, bytes, false, what));
        const int where = place(p, what);
        if (where < 0) return where;
        if (where) {
            *out = p;
            return 0;
        }
        LN_REQUIRE(!capturing, "%s is a host array: a captured call takes device memory only", what);
        void* d;
        LN_TRY(transform_ws(ctx, ws, bytes, &d));
        LN_HIP(hipMemcpyAsync(d, p, bytes, hipMemcpyHostToDevice, ctx->stream));
        *out = d;
        return 0;
    }
    // keep: the call may leave parts of it as they were
    int out(void* p, size_t bytes, int ws, bool keep, const char* what, void** dev) {
        *dev = nullptr;
        if (!p || bytes == 0) return 0;
        LN_TRY(note(p, bytes, true, what));
        const int where = place(p, what);
        if (where < 0) return where;
        if (where) {
            *dev = p;
            return 0;
        }
        LN_REQUIRE(!capturing, "%s is a host array: a captured call takes device memory only", what);
        LN_TRY(transform_ws(ctx, ws, bytes, dev));
        if (keep) LN_HIP(hipMemcpyAsync(*dev, p, bytes, hipMemcpyHostToDevice, ctx->stream));
        back[nback++] = {p, *dev, bytes};
        return 0;
    }
    int finish() {
        for (int i = 0; i < nback; ++i) LN_HIP(hipMemcpyAsync(back[i].host, back[i].dev, back[i].bytes, hipMemcpyDeviceToHost, ctx->stream));
        // copies from pinned memory run later: the caller may change it once the call has returned
        if (nback || pinned) LN_HIP(hipStreamSynchronize(ctx->stream));
        return 0;
    }
};

constexpr int kMaxWidth = 1 << 20;

int check_matrix(const char* what, int64_t rows, int cols, int64_t ld) {
    LN_REQUIRE(rows <= 1 || ld >= cols, "%s: row stride %lld under its width %d", what, (long long)ld, cols);
    LN_REQUIRE(ld < (1ll << 40), "%s: row stride %lld", what, (long long)ld);
    return 0;
}
size_t matrix_bytes(int64_t rows, int cols, int64_t ld, size_t e) { return rows ? ((size_t)(rows - 1) * ld + cols) * e : 0; }

// offsets and slots of a call; *covered: the host knows that every row belongs to a segment (with a group, if `need_group`)
int segments(Call& c, const int64_t* offsets, const int32_t* slots, int S, int G, int64_t rows, bool need_group, Segments* sg, bool* covered) {
    LN_REQUIRE(S >= 0 && G >= 0 && rows >= 0, "negative size: %d segments, %d groups, %lld rows", S, G, (long long)rows);
    LN_REQUIRE(rows < (1ll << 40), "%lld rows", (long long)rows);
    LN_REQUIRE(S == 0 || offsets, "offsets is null");
    // (no segments: an empty array of slots may well be a null pointer)
    LN_REQUIRE(slots || S == G || S == 0, "%d segments of %d groups: without slots there is one segment for each group", S, G);
    *covered = rows == 0;
    *sg = Segments{nullptr, nullptr, S, G, rows};
    if (S == 0) return 0;
    const int where = c.place(offsets, "offsets");
    if (where < 0) return where;
    bool known = where == 0;
    if (where == 0) {
        LN_REQUIRE(offsets[0] >= 0 && offsets[S] <= rows, "offsets run from %lld to %lld, there are %lld rows", (long long)offsets[0],
                   (long long)offsets[S], (long long)rows);
        for (int s = 0; s < S; ++s)
            LN_REQUIRE(offsets[s] <= offsets[s + 1], "offsets fall from %lld to %lld at segment %d", (long long)offsets[s],
                       (long long)offsets[s + 1], s);
        known = offsets[0] == 0 && offsets[S] == rows;
    }
    const void* d;
    LN_TRY(c.in(offsets, (size_t)(S + 1) * 8, kTrOff, "offsets", &d));
    sg->off = (const int64_t*)d;
    if (slots) {
        const int ws = c.place(slots, "slots");
        if (ws < 0) return ws;
        if (ws == 0)
            for (int s = 0; s < S; ++s)
                LN_REQUIRE(slots[s] < G && slots[s] >= (need_group ? 0 : -1), "slots[%d] = %d, there are %d groups", s, slots[s], G);
        else if (need_group)
            known = false;
        LN_TRY(c.in(slots, (size_t)S * 4, kTrSlots, "slots", &d));
        sg->slots = (const int32_t*)d;
    }
    *covered = known || rows == 0;
    return 0;
}

int check_type(int dtype) {
    LN_REQUIRE(dtype == LNASR_F64 || dtype == LNASR_F32 || dtype == LNASR_F16 || dtype == LNASR_BF16, "dtype %d", dtype);
    return 0;
}

}  // namespace
}  // namespace lnasr

using namespace lnasr;

extern "C" {

int lnasr_affine(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets, const int32_t* slots,
                 int S, const void* w, const void* bias, int G, int dout, void* y, int64_t ldy) try {
    LN_REQUIRE(ctx, "null ctx");
    DeviceScope scope(ctx);
    LN_HIP(hipSetDevice(ctx->device));
    LN_TRY(check_type(dtype));
    LN_REQUIRE(din > 0 && dout > 0 && din <= kMaxWidth && dout <= kMaxWidth, "widths %d -> %d", din, dout);
    LN_TRY(check_matrix("x", rows, din, ldx));
    LN_TRY(check_matrix("y", rows, dout, ldy));
    const size_t e = transform_size(dtype);
    Call c(ctx);
    LN_TRY(c.begin());
    Segments sg;
    bool covered;
    LN_TRY(segments(c, offsets, slots, S, G, rows, true, &sg, &covered));
    LN_REQUIRE(G > 0 || S == 0, "no transforms for %d segments", S);
    if (rows == 0 || S == 0) return 0;
    LN_REQUIRE(y, "y is null");
    RowsArgs a{};
    a.sg = sg;
    LN_TRY(c.in(x, matrix_bytes(rows, din, ldx, e), kTrX, "x", &a.x));
    LN_TRY(c.in(w, (size_t)G * dout * din * e, kTrW, "w", &a.w));
    if (bias) LN_TRY(c.in(bias, (size_t)G * dout * e, kTrBias, "bias", &a.bias));
    LN_TRY(c.out(y, matrix_bytes(rows, dout, ldy, e), kTrOut0, !covered || ldy != dout, "y", &a.y));
    a.ldx = ldx;
    a.ldy = ldy;
    a.w_stride = (int64_t)dout * din;
    a.bias_stride = dout;
    a.K = din;
    a.N = dout;
    LN_TRY(transform_rows(ctx, dtype, a, "affine"));
    return c.finish();
} catch (const std::exception& e) {
    return fail(LNASR_E_INVALID, "%s", e.what());
}

int lnasr_affine_grad(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                      const int32_t* slots, int S, const void* w, int G, int dout, const void* dy, int64_t lddy, void* dx, int64_t lddx,
                      void* dw, void* dbias) try {
    LN_REQUIRE(ctx, "null ctx");
    DeviceScope scope(ctx);
    LN_HIP(hipSetDevice(ctx->device));
    LN_TRY(check_type(dtype));
    LN_REQUIRE(din > 0 && dout > 0 && din <= kMaxWidth && dout <= kMaxWidth, "widths %d -> %d", din, dout);
    LN_TRY(check_matrix("x", rows, din, dw ? ldx : din));
    LN_TRY(check_matrix("dy", rows, dout, lddy));
    LN_TRY(check_matrix("dx", rows, din, dx ? lddx : din));
    LN_REQUIRE(!dbias || dw, "the gradient of bias comes with that of w");
    const size_t e = transform_size(dtype);
    Call c(ctx);
    LN_TRY(c.begin());
    Segments sg;
    bool covered;
    LN_TRY(segments(c, offsets, slots, S, G, rows, true, &sg, &covered));
    LN_REQUIRE(G > 0 || S == 0, "no transforms for %d segments", S);
    if (G == 0) return 0;
    const void *d_x = nullptr, *d_w = nullptr, *d_dy = nullptr;
    void *d_dx, *d_dw, *d_db;
    LN_TRY(c.in(dy, matrix_bytes(rows, dout, lddy, e), kTrDy, "dy", &d_dy));
    if (dw) LN_TRY(c.in(x, matrix_bytes(rows, din, ldx, e), kTrX, "x", &d_x));
    if (dx) LN_TRY(c.in(w, (size_t)G * dout * din * e, kTrW, "w", &d_w));
    LN_TRY(c.out(dx, matrix_bytes(rows, din, lddx, e), kTrOut0, !covered || lddx != din, "dx", &d_dx));
    LN_TRY(c.out(dw, (size_t)G * dout * din * e, kTrOut1, false, "dw", &d_dw));
    LN_TRY(c.out(dbias, (size_t)G * dout * e, kTrOut2, false, "dbias", &d_db));
    if (d_dx) {
        RowsArgs a{};
        a.sg = sg;
        a.x = d_dy;
        a.ldx = lddy;
        a.w = d_w;
        a.w_stride = (int64_t)dout * din;
        a.y = d_dx;
        a.ldy = lddx;
        a.K = dout;
        a.N = din;
        a.kn = true;
        LN_TRY(transform_rows(ctx, dtype, a, "affine_dx"));
    }
    if (d_dw) {
        SumArgs a{};
        a.sg = sg;
        a.group_step = 1;
        a.groups = G;
        LN_TRY(transform_sort(ctx, std::max(ldx, lddy), &a));
        a.a = d_dy;
        a.lda = lddy;
        a.I = dout;
        a.b = d_x;
        a.ldb = ldx;
        a.J = din;
        a.out = d_dw;
        a.cols = d_db;
        LN_TRY(transform_sum(ctx, dtype, a, "affine_dw"));
    }
    return c.finish();
} catch (const std::exception& e) {
    return fail(LNASR_E_INVALID, "%s", e.what());
}

int lnasr_projection(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                     const int32_t* slots, int S, const void* w, const void* bias, int dout, const void* a, const void* b,
                     const double* scale, int G, int rank, void* y, int64_t ldy) try {
    LN_REQUIRE(ctx, "null ctx");
    DeviceScope scope(ctx);
    LN_HIP(hipSetDevice(ctx->device));
    LN_TRY(check_type(dtype));
    LN_REQUIRE(din > 0 && dout > 0 && din <= kMaxWidth && dout <= kMaxWidth, "widths %d -> %d", din, dout);
    LN_REQUIRE(rank > 0 && rank <= kMaxWidth, "rank %d", rank);
    LN_TRY(check_matrix("x", rows, din, ldx));
    LN_TRY(check_matrix("y", rows, dout, ldy));
    const size_t e = transform_size(dtype);
    Call c(ctx);
    LN_TRY(c.begin());
    Segments sg;
    bool covered;
    LN_TRY(segments(c, offsets, slots, S, G, rows, false, &sg, &covered));
    if (rows == 0 || S == 0) return 0;
    LN_REQUIRE(y, "y is null");
    RowsArgs m{}, low{};
    LN_TRY(c.in(x, matrix_bytes(rows, din, ldx, e), kTrX, "x", &m.x));
    LN_TRY(c.in(w, (size_t)dout * din * e, kTrW, "w", &m.w));
    if (bias) LN_TRY(c.in(bias, (size_t)dout * e, kTrBias, "bias", &m.bias));
    LN_TRY(c.in(a, (size_t)G * rank * din * e, kTrA, "a", &low.w));
    LN_TRY(c.in(b, (size_t)G * dout * rank * e, kTrB, "b", &m.low));
    if (scale) LN_TRY(c.in(scale, (size_t)G * 8, kTrScale, "scale", (const void**)&low.scale));
    LN_TRY(c.out(y, matrix_bytes(rows, dout, ldy, e), kTrOut0, !covered || ldy != dout, "y", &m.y));
    m.sg = low.sg = sg;
    m.ldx = low.ldx = ldx;
    m.ldy = ldy;
    m.K = low.K = din;
    m.N = dout;
    if (G > 0) {
        // the narrow middle, held in 32 bits or more, rows padded to whole 16-byte pieces
        const size_t me = transform_mid_size(dtype);
        const int64_t ldp = (rank * me + 15) / 16 * 16 / me;
        void* p;
        LN_TRY(transform_ws(ctx, kTrLow, (size_t)rows * ldp * me, &p));
        low.mid = true;
        low.x = m.x;
        low.w_stride = (int64_t)rank * din;
        low.y = p;
        low.ldy = ldp;
        low.N = rank;
        LN_TRY(transform_rows(ctx, dtype, low, "projection_low"));
        m.p = p;
        m.ldp = ldp;
        m.R = rank;
        m.low_stride = (int64_t)dout * rank;
    } else {
        m.low = nullptr;
    }
    LN_TRY(transform_rows(ctx, dtype, m, "projection"));
    return c.finish();
} catch (const std::exception& e) {
    return fail(LNASR_E_INVALID, "%s", e.what());
}

int lnasr_projection_grad(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                          const int32_t* slots, int S, const void* w, int dout, const void* a, const void* b, const double* scale, int G,
                          int rank, const void* dy, int64_t lddy, void* dx, int64_t lddx, void* da, void* db, void* dw, void* dbias) try {
    LN_REQUIRE(ctx, "null ctx");
    DeviceScope scope(ctx);
    LN_HIP(hipSetDevice(ctx->device));
    LN_TRY(check_type(dtype));
    LN_REQUIRE(din > 0 && dout > 0 && din <= kMaxWidth && dout <= kMaxWidth, "widths %d -> %d", din, dout);
    LN_REQUIRE(rank > 0 && rank <= kMaxWidth, "rank %d", rank);
    const bool need_x = da || db || dw;
    LN_TRY(check_matrix("x", rows, din, need_x ? ldx : din));
    LN_TRY(check_matrix("dy", rows, dout, lddy));
    LN_TRY(check_matrix("dx", rows, din, dx ? lddx : din));
    LN_REQUIRE(!dbias || dw, "the gradient of bias comes with that of w");
    const size_t e = transform_size(dtype);
    Call c(ctx);
    LN_TRY(c.begin());
    Segments sg;
    bool covered;
    LN_TRY(segments(c, offsets, slots, S, G, rows, false, &sg, &covered));
    const void *d_x = nullptr, *d_w = nullptr, *d_a = nullptr, *d_b = nullptr, *d_dy = nullptr;
    const double* d_scale = nullptr;
    void *d_dx, *d_da, *d_db, *d_dw, *d_dbias, *p = nullptr, *dp = nullptr;
    LN_TRY(c.in(dy, matrix_bytes(rows, dout, lddy, e), kTrDy, "dy", &d_dy));
    if (need_x) LN_TRY(c.in(x, matrix_bytes(rows, din, ldx, e), kTrX, "x", &d_x));
    if (dx) LN_TRY(c.in(w, (size_t)dout * din * e, kTrW, "w", &d_w));
    if (dx || db) LN_TRY(c.in(a, (size_t)G * rank * din * e, kTrA, "a", &d_a));
    if (dx || da) LN_TRY(c.in(b, (size_t)G * dout * rank * e, kTrB, "b", &d_b));
    if (scale) LN_TRY(c.in(scale, (size_t)G * 8, kTrScale, "scale", (const void**)&d_scale));
    LN_TRY(c.out(dx, matrix_bytes(rows, din, lddx, e), kTrOut0, !covered || lddx != din, "dx", &d_dx));
    LN_TRY(c.out(da, (size_t)G * rank * din * e, kTrOut1, false, "da", &d_da));
    LN_TRY(c.out(db, (size_t)G * dout * rank * e, kTrOut2, false, "db", &d_db));
    LN_TRY(c.out(dw, (size_t)dout * din * e, kTrOut3, false, "dw", &d_dw));
    LN_TRY(c.out(dbias, (size_t)dout * e, kTrOut4, false, "dbias", &d_dbias));
    const size_t me = transform_mid_size(dtype);
    const int64_t ldp = (rank * me + 15) / 16 * 16 / me;
    RowsArgs r{};
    r.sg = sg;
    r.mid = true;
    r.scale = d_scale;
    r.ldy = ldp;
    r.N = rank;
    r.w_stride = (int64_t)rank * din;
    if (G > 0 && (d_dx || d_da)) {                       // scale_k B_k^T dy
        LN_TRY(transform_ws(ctx, kTrDlow, (size_t)rows * ldp * me, &dp));
        r.x = d_dy;
        r.ldx = lddy;
        r.K = dout;
        r.w = d_b;
        r.w_stride = (int64_t)dout * rank;
        r.y = dp;
        r.kn = true;
        LN_TRY(transform_rows(ctx, dtype, r, "projection_dlow"));
    }
    if (d_db) {                                          // scale_k A_k x
        LN_TRY(transform_ws(ctx, kTrLow, (size_t)rows * ldp * me, &p));
        r.x = d_x;
        r.ldx = ldx;
        r.K = din;
        r.w = d_a;
        r.w_stride = (int64_t)rank * din;
        r.y = p;
        r.kn = false;
        LN_TRY(transform_rows(ctx, dtype, r, "projection_low"));
    }
    if (d_dx && S > 0) {
        RowsArgs m{};
        m.sg = sg;
        m.x = d_dy;
        m.ldx = lddy;
        m.w = d_w;
        m.y = d_dx;
        m.ldy = lddx;
        m.K = dout;
        m.N = din;
        m.kn = true;
        if (G > 0) {
            m.p = dp;
            m.ldp = ldp;
            m.low = d_a;
            m.low_stride = (int64_t)rank * din;
            m.R = rank;
        }
        LN_TRY(transform_rows(ctx, dtype, m, "projection_dx"));
    }
    SumArgs t{};
    t.sg = sg;
    if (d_da || d_db) {
        t.group_step = 1;
        t.groups = G;
        if (S > 0) LN_TRY(transform_sort(ctx, std::max(ldx, lddy), &t));
    }
    if (d_da) {
        t.a = dp;
        t.lda = ldp;
        t.I = rank;
        t.b = d_x;
        t.ldb = ldx;
        t.J = din;
        t.mid_a = true;
        t.out = d_da;
        LN_TRY(transform_sum(ctx, dtype, t, "projection_da"));
    }
    if (d_db) {
        t.a = d_dy;
        t.lda = lddy;
        t.I = dout;
        t.b = p;
        t.ldb = ldp;
        t.J = rank;
        t.mid_a = false;
        t.mid_b = true;
        t.out = d_db;
        LN_TRY(transform_sum(ctx, dtype, t, "projection_db"));
    }
    if (d_dw) {
        SumArgs s{};
        s.sg = sg;
        s.group_off = sg.off;
        s.group_step = S;
        s.groups = 1;
        s.a = d_dy;
        s.lda = lddy;
        s.I = dout;
        s.b = d_x;
        s.ldb = ldx;
        s.J = din;
        s.out = d_dw;
        s.cols = d_dbias;
        LN_TRY(transform_sum(ctx, dtype, s, "projection_dw"));
    }
    return c.finish();
} catch (const std::exception& e) {
    return fail(LNASR_E_INVALID, "%s", e.what());
}

}  // extern "C"
