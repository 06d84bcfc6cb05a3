// devops_capi.cpp — the flat C ABI of the operators in devops.h: argument checks, streams and
// workspaces.  Every entry returns 0 or a negative code (include/ggml-mi355x.h) and launches
// nothing when it refuses; none aborts or throws.
#include "devops.h"

#include "../../include/ggml-mi355x.h"

using namespace mi355x_ops;

#define OPS_API extern "C" __attribute__((visibility("default")))

namespace {

// NULL: a private stream, waited for before the call returns; MI355X_STREAM_DEFAULT: the device's
// default stream; anything else as it is, not waited for
struct call_stream {
    hipStream_t st = nullptr;
    bool own = false;
    hipError_t err = hipSuccess;
    explicit call_stream(void * s) {
        if (s == MI355X_STREAM_DEFAULT) return;
        if (s) {
            st = (hipStream_t) s;
        } else {
            err = hipStreamCreateWithFlags(&st, hipStreamNonBlocking);
            own = err == hipSuccess;
        }
    }
    ~call_stream() {
        if (own) (void) hipStreamDestroy(st);
    }
    // after a failed launch too: one in front of it may still be at work on the caller's memory
    int done(hipError_t e) {
        const hipError_t waited = own ? hipStreamSynchronize(st) : hipSuccess;
        return e == hipSuccess && waited == hipSuccess ? 0 : MI355X_ERR_HIP;
    }
};

bool is_elem(int t) { return t == ELEM_F32 || t == ELEM_F16 || t == ELEM_BF16; }
int64_t elem_size(int t) { return t == ELEM_F32 ? 4 : 2; }
bool aligned(const void * p, uintptr_t n) { return (uintptr_t) p % n == 0; }

// where there is something to do, a pointer that the call needs is not NULL
template <class... P> int present(const P *... p) { return ((p != nullptr) && ...) ? 0 : MI355X_ERR_SHAPE; }

constexpr int64_t MAX_K = (int64_t) 1 << 24;       // elements of a row
constexpr int64_t MAX_ROWS = (int64_t) 1 << 31;    // rows of a matrix, pairs of a routing step (exclusive)

int check_rows(int64_t rows, int64_t K) {
    if (rows < 0 || rows >= MAX_ROWS) return MI355X_ERR_SHAPE;
    if (K <= 0 || K % MX4_BLOCK || K > MAX_K) return MI355X_ERR_SHAPE;
    return 0;
}

// codes are read 16 bytes at a time, exponents 8
int check_mx4(const void * codes, const void * scales) {
    return aligned(codes, 16) && aligned(scales, 8) ? 0 : MI355X_ERR_ALIGN;
}

int check_elems(int type, const void * p) {
    if (!is_elem(type)) return MI355X_ERR_TYPE;
    return aligned(p, (uintptr_t) elem_size(type)) ? 0 : MI355X_ERR_ALIGN;
}

// integers and float32 weights, in as many arrays as the call has
template <class... P> int check_words(const P *... p) { return (aligned(p, 4) && ...) ? 0 : MI355X_ERR_ALIGN; }

int check_routing(int64_t T, int64_t used) {
    if (used <= 0 || used > MOE_MAX_USED || T < 0 || T >= MAX_ROWS || T * used >= MAX_ROWS) return MI355X_ERR_SHAPE;
    return 0;
}

int64_t codes_bytes(int64_t rows, int64_t K) { return (rows * (K / 2) + 255) / 256 * 256; }
int64_t scales_bytes(int64_t rows, int64_t K) { return (K + MX4_PLANE - 1) / MX4_PLANE * rows * 8; }

#define TRY(expr)                    \
    do {                             \
        const int rc_ = (expr);      \
        if (rc_) return rc_;         \
    } while (0)

}  // namespace

OPS_API int64_t mi355x_mx4_scales_bytes(int64_t rows, int64_t K) { return check_rows(rows, K) ? -1 : scales_bytes(rows, K); }

OPS_API int mi355x_mx4_quantize(int xtype, const void * x, int64_t ldx, int64_t rows, int64_t K, uint8_t * codes,
                                uint8_t * scales, void * stream) {
    TRY(check_rows(rows, K));
    TRY(check_elems(xtype, x));
    TRY(check_mx4(codes, scales));
    if (ldx < K && rows > 1) return MI355X_ERR_SHAPE;
    if (rows == 0) return 0;
    TRY(present(x, codes, scales));
    call_stream cs(stream);
    if (cs.err != hipSuccess) return MI355X_ERR_HIP;
    return cs.done(mx4_quantize(xtype, x, ldx, rows, K, codes, scales, cs.st));
}

OPS_API int mi355x_mx4_dequantize(const uint8_t * codes, const uint8_t * scales, int64_t rows, int64_t K, int ytype, void * y,
                                  void * stream) {
    TRY(check_rows(rows, K));
    TRY(check_elems(ytype, y));
    TRY(check_mx4(codes, scales));
    if (rows == 0) return 0;
    TRY(present(codes, scales, y));
    call_stream cs(stream);
    if (cs.err != hipSuccess) return MI355X_ERR_HIP;
    return cs.done(mx4_dequantize({codes, scales, rows, K}, ytype, y, cs.st));
}

// a product's arguments, checked; x_rows rows of x
struct product {
    mx4_mat w;
    int xtype;
    const void * x;
    const uint8_t * x_scales;
    int64_t ldx, x_rows;
    const moe_view * view;
    int ytype;
    void * y;

    int64_t x_bytes() const { return codes_bytes(x_rows, w.K) + (scales_bytes(x_rows, w.K) + 255) / 256 * 256; }

    int64_t workspace() const {
        const mx4_needs n = mx4_product_needs(w, x_rows, view);
        return (xtype != MI355X_MX4 && n.quantized ? x_bytes() : 0) + n.part;
    }

    int check_shape() const {
        TRY(check_rows(w.rows, w.K));
        TRY(check_rows(x_rows, w.K));
        return xtype == MI355X_MX4 || is_elem(xtype) ? 0 : MI355X_ERR_TYPE;
    }

    int run(void * work, int64_t work_bytes, void * stream) const {
        TRY(check_shape());
        TRY(check_mx4(w.codes, w.scales));
        if (xtype == MI355X_MX4) TRY(check_mx4(x, x_scales));
        else TRY(check_elems(xtype, x));
        if (xtype != MI355X_MX4 && ldx < w.K && x_rows > 1) return MI355X_ERR_SHAPE;
        TRY(check_elems(ytype, y));
        if (view) TRY(check_words(view->order, view->offsets));
        if (!aligned(work, 16)) return MI355X_ERR_ALIGN;
        if (x_rows == 0 || w.rows == 0) return 0;
        TRY(present(w.codes, w.scales, x, y));
        if (xtype == MI355X_MX4) TRY(present(x_scales));
        if (view) TRY(present(view->order, view->offsets));
        const int64_t needed = workspace();
        if (work_bytes < needed || (needed && !work)) return MI355X_ERR_WORKSPACE;
        call_stream cs(stream);
        if (cs.err != hipSuccess) return MI355X_ERR_HIP;
        if (xtype == MI355X_MX4)
            return cs.done(mx4_product(w, {(const uint8_t *) x, x_scales, x_rows, w.K}, view, ytype, y, work, cs.st));
        if (!mx4_product_needs(w, x_rows, view).quantized)
            return cs.done(mx4_product_float(w, xtype, x, ldx, x_rows, view, ytype, y, cs.st));
        uint8_t * codes = (uint8_t *) work, * scales = codes + codes_bytes(x_rows, w.K);
        const hipError_t e = mx4_quantize(xtype, x, ldx, x_rows, w.K, codes, scales, cs.st);
        if (e != hipSuccess) return cs.done(e);
        return cs.done(mx4_product(w, {codes, scales, x_rows, w.K}, view, ytype, y, codes + x_bytes(), cs.st));
    }
};

static int check_experts(int64_t n_expert) { return n_expert > 0 && n_expert <= MOE_MAX_EXPERTS ? 0 : MI355X_ERR_SHAPE; }

OPS_API int64_t mi355x_mx4_mul_mat_workspace(int64_t M, int64_t K, int xtype, int64_t T) {
    const product p = {{nullptr, nullptr, M, K}, xtype, nullptr, nullptr, K, T, nullptr, ELEM_F32, nullptr};
    return p.check_shape() ? -1 : T == 0 || M == 0 ? 0 : p.workspace();
}

OPS_API int mi355x_mx4_mul_mat(const uint8_t * w_codes, const uint8_t * w_scales, int64_t M, int64_t K, int xtype,
                               const void * x, const uint8_t * x_scales, int64_t ldx, int64_t T, int ytype, void * y,
                               void * work, int64_t work_bytes, void * stream) {
    const product p = {{w_codes, w_scales, M, K}, xtype, x, x_scales, ldx, T, nullptr, ytype, y};
    return p.run(work, work_bytes, stream);
}

OPS_API int64_t mi355x_mx4_mul_mat_id_workspace(int64_t M, int64_t K, int64_t n_expert, int xtype, int64_t T, int64_t used,
                                                int x_sorted) {
    if (check_routing(T, used) || check_experts(n_expert)) return -1;
    const moe_view v = {nullptr, nullptr, T * used, (int) n_expert, x_sorted ? 0 : (int) used};
    const product p = {{nullptr, nullptr, M, K}, xtype, nullptr, nullptr, K, x_sorted ? T * used : T, &v, ELEM_F32, nullptr};
    return p.check_shape() ? -1 : T == 0 || M == 0 ? 0 : p.workspace();
}

OPS_API int mi355x_mx4_mul_mat_id(const uint8_t * w_codes, const uint8_t * w_scales, int64_t M, int64_t K, int64_t n_expert,
                                  int xtype, const void * x, const uint8_t * x_scales, int64_t ldx, int64_t T, int64_t used,
                                  int x_sorted, const int32_t * order, const int32_t * offsets, int ytype, void * y,
                                  void * work, int64_t work_bytes, void * stream) {
    TRY(check_routing(T, used));
    TRY(check_experts(n_expert));
    const moe_view v = {order, offsets, T * used, (int) n_expert, x_sorted ? 0 : (int) used};
    const product p = {{w_codes, w_scales, M, K}, xtype, x, x_scales, ldx, x_sorted ? T * used : T, &v, ytype, y};
    return p.run(work, work_bytes, stream);
}

OPS_API int64_t mi355x_moe_sort_workspace(int64_t T, int64_t used, int64_t n_expert) {
    if (check_routing(T, used) || n_expert <= 0 || n_expert > MOE_MAX_EXPERTS) return -1;
    return (int64_t) moe_sort_workspace(T * used, (int) n_expert);
}

OPS_API int mi355x_moe_sort(const void * ids, int id_bytes, int64_t T, int64_t used, int64_t n_expert, int32_t * order,
                            int32_t * rank, int32_t * offsets, void * work, int64_t work_bytes, void * stream) {
    TRY(check_routing(T, used));
    if (n_expert <= 0 || n_expert > MOE_MAX_EXPERTS) return MI355X_ERR_SHAPE;
    if (id_bytes != 4 && id_bytes != 8) return MI355X_ERR_TYPE;
    if (!aligned(ids, id_bytes) || !aligned(work, 4)) return MI355X_ERR_ALIGN;
    TRY(check_words(order, rank, offsets));
    TRY(present(offsets));
    if (T > 0) TRY(present(ids, order, rank));
    const int64_t needed = (int64_t) moe_sort_workspace(T * used, (int) n_expert);
    if (work_bytes < needed || (needed && !work)) return MI355X_ERR_WORKSPACE;
    call_stream cs(stream);
    if (cs.err != hipSuccess) return MI355X_ERR_HIP;
    return cs.done(moe_sort(ids, id_bytes, T * used, (int) n_expert, order, rank, offsets, work, cs.st));
}

OPS_API int mi355x_moe_gather(int type, const void * x, int64_t ldx, int64_t T, int64_t D, int64_t used, const int32_t * order,
                              const int32_t * rank, void * xs, void * stream) {
    TRY(check_routing(T, used));
    TRY(check_elems(type, x));
    TRY(check_elems(type, xs));
    TRY(check_words(order, rank));
    if (D < 0 || D > MAX_K || (ldx < D && T > 1)) return MI355X_ERR_SHAPE;
    if (T == 0 || D == 0) return 0;
    TRY(present(x, order, rank, xs));
    call_stream cs(stream);
    if (cs.err != hipSuccess) return MI355X_ERR_HIP;
    return cs.done(moe_gather(type, x, ldx, T, D, (int) used, order, rank, xs, cs.st));
}

OPS_API int mi355x_moe_combine(int type, const void * ys, int64_t ldys, int64_t T, int64_t D, int64_t used,
                               const int32_t * rank, const float * w, void * y, void * stream) {
    TRY(check_routing(T, used));
    TRY(check_elems(type, ys));
    TRY(check_elems(type, y));
    TRY(check_words(rank, w));
    if (D < 0 || D > MAX_K || (ldys < D && T * used > 1)) return MI355X_ERR_SHAPE;
    if (T == 0 || D == 0) return 0;
    TRY(present(ys, rank, y));   // w may be NULL
    call_stream cs(stream);
    if (cs.err != hipSuccess) return MI355X_ERR_HIP;
    return cs.done(moe_combine(type, ys, ldys, T, D, (int) used, rank, w, y, cs.st));
}

OPS_API int mi355x_moe_combine_back(int type, const void * dy, int64_t lddy, const void * ys, int64_t ldys, int64_t T,
                                    int64_t D, int64_t used, const int32_t * order, const int32_t * rank, const float * w,
                                    void * dys, float * dw, void * stream) {
    TRY(check_routing(T, used));
    TRY(check_elems(type, dy));
    TRY(check_elems(type, ys));
    TRY(check_elems(type, dys));
    TRY(check_words(order, rank, w, dw));
    if (D < 0 || D > MAX_K || (lddy < D && T > 1) || (ldys < D && T * used > 1)) return MI355X_ERR_SHAPE;
    if (T == 0) return 0;
    TRY(present(order, rank, w, dw));
    if (D > 0) TRY(present(dy, ys, dys));
    call_stream cs(stream);
    if (cs.err != hipSuccess) return MI355X_ERR_HIP;
    return cs.done(moe_combine_back(type, dy, lddy, ys, ldys, T, D, (int) used, order, rank, w, dys, dw, cs.st));
}
