// devops_torch.cpp — the Python binding of the operators in include/ggml-mi355x.h: torch tensors in,
// torch tensors out, on the tensors' device and torch's current stream of it.  In C++ because the
// smallest calls last a few microseconds on the device, less than argument handling takes in Python.
// llamacog_amd/device_ops.py documents the functions; here are the checks, the output allocations
// and the calls.
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>

#include "../../include/ggml-mi355x.h"

using at::Tensor;

namespace {

// ---- checks ----------------------------------------------------------------------------------
const char * const ELEMS = "float32, float16 or bfloat16 is wanted, got ";

int elem_type(at::ScalarType t, const char * what) {
    switch (t) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 30;
        default: TORCH_CHECK_TYPE(false, what, ": ", ELEMS, t);
    }
}

void on_gpu(const Tensor & t, const char * what) {
    TORCH_CHECK_VALUE(t.is_cuda(), what, ": a tensor on an MI355X is wanted, got one on ", t.device());
}

void beside(const Tensor & t, const char * what, const Tensor & other) {
    on_gpu(t, what);
    TORCH_CHECK_VALUE(t.device() == other.device(), what, ": on ", t.device(), ", the others on ", other.device());
}

// neither a gradient is recorded nor a tangent passed on (forward mode, which no_grad() leaves on)
void no_gradient(const Tensor & t, const char * what) {
    TORCH_CHECK_VALUE(!t.requires_grad() || !at::GradMode::is_enabled(), what,
                      ": no gradient is recorded here; pass a detached tensor");
    TORCH_CHECK_VALUE(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), what,
                      ": no tangent is passed on here; pass a tensor without one");
}

// its memory holds the values: not a view that negates them
void plain(const Tensor & t, const char * what) {
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && !t.is_neg(), what, ": a strided tensor that is no lazily negated view is wanted");
}

// a float [rows, columns] tensor whose columns lie side by side and whose rows do not overlap; returns its type
int matrix(const Tensor & t, const char * what) {
    no_gradient(t, what);
    on_gpu(t, what);
    const int type = elem_type(t.scalar_type(), what);
    plain(t, what);
    TORCH_CHECK_VALUE(t.dim() == 2, what, ": [rows, columns] is wanted, got ", t.sizes());
    TORCH_CHECK_VALUE((t.stride(1) == 1 || t.size(1) <= 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)), what,
                      ": columns have to lie side by side and rows apart, got strides ", t.strides());
    return type;
}

// elements from one row to the next, for a single row its length
int64_t row_step(const Tensor & t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void whole(const Tensor & t, const char * what, const Tensor & other, at::ScalarType type, at::IntArrayRef shape) {
    beside(t, what, other);
    plain(t, what);
    TORCH_CHECK_TYPE(t.scalar_type() == type, what, ": ", type, " is wanted, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.sizes() == shape && t.is_contiguous(), what, ": a contiguous tensor of shape ", shape,
                      " is wanted, got ", t.sizes(), ", strides ", t.strides());
}

void whole_blocks(int64_t k, const char * what) {
    TORCH_CHECK_VALUE(k > 0 && k % 32 == 0, what, ": rows of a multiple of 32 elements are wanted, got ", k);
}

struct mx4 {
    int64_t rows, k;
};

mx4 check_mx4(const Tensor & codes, const Tensor & scales, const char * what, int dims) {
    on_gpu(codes, what);
    plain(codes, what);
    TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte, what, ".codes: uint8 is wanted, got ", codes.scalar_type());
    TORCH_CHECK_VALUE(codes.dim() == dims && codes.is_contiguous(), what, ".codes: a contiguous tensor of ", dims,
                      " dimensions is wanted, got ", codes.sizes(), ", strides ", codes.strides());
    const mx4 m = {codes.size(-2), codes.size(-1) * 2};
    whole_blocks(m.k, what);
    const int64_t planes = (m.k + 255) / 256;
    if (dims == 3) whole(scales, "scales", codes, at::kByte, {codes.size(0), planes, m.rows, 8});
    else whole(scales, "scales", codes, at::kByte, {planes, m.rows, 8});
    return m;
}

struct plan {
    int64_t t, used, experts;
};

void check_routing(int64_t used, int64_t experts) {
    TORCH_CHECK_VALUE(used >= 1 && used <= 16, "1 to 16 slots per token are supported, got ", used);
    TORCH_CHECK_VALUE(experts >= 1 && experts <= 1024, "1 to 1024 experts are supported, got ", experts);
}

plan check_plan(const Tensor & order, const Tensor & rank, const Tensor & offsets, const Tensor & other) {
    TORCH_CHECK_VALUE(rank.dim() == 2 && offsets.dim() == 1, "plan: rank [T, used] and offsets [n_expert + 1] are wanted");
    const plan p = {rank.size(0), rank.size(1), offsets.size(0) - 1};
    check_routing(p.used, p.experts);
    whole(rank, "plan.rank", other, at::kInt, {p.t, p.used});
    whole(order, "plan.order", other, at::kInt, {p.t * p.used});
    whole(offsets, "plan.offsets", other, at::kInt, {p.experts + 1});
    return p;
}

// ---- calls -----------------------------------------------------------------------------------
// the tensors' device as the current one, and torch's current stream of it
struct launch {
    c10::DeviceIndex before, device;
    void * stream;
    explicit launch(const Tensor & t) : before(c10::hip::current_device()), device(t.device().index()) {
        if (device != before) c10::hip::set_device(device);
        stream = c10::hip::getCurrentHIPStream(device).stream();
        if (!stream) stream = MI355X_STREAM_DEFAULT;   // NULL is a private stream there
    }
    ~launch() {
        if (device != before) c10::hip::set_device(before);
    }
};

void check(int rc, const char * what) {
    if (rc == 0) return;
    TORCH_CHECK_TYPE(rc != MI355X_ERR_TYPE, what, ": unsupported element type");
    TORCH_CHECK_VALUE(rc != MI355X_ERR_SHAPE, what, ": unsupported shape");
    TORCH_CHECK_VALUE(rc != MI355X_ERR_ALIGN, what, ": misaligned tensor");
    TORCH_CHECK(false, what, rc == MI355X_ERR_WORKSPACE ? ": workspace too small" : ": HIP error");
}

const uint8_t * bytes(const Tensor & t) { return (const uint8_t *) t.const_data_ptr(); }
const int32_t * ints(const Tensor & t) { return (const int32_t *) t.const_data_ptr(); }

Tensor fresh(at::IntArrayRef shape, const Tensor & like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type)); }

std::tuple<Tensor, Tensor> quantize(const Tensor & x) {
    const int type = matrix(x, "x");
    const int64_t rows = x.size(0), k = x.size(1);
    whole_blocks(k, "x");
    Tensor codes = fresh({rows, k / 2}, x, at::kByte), scales = fresh({(k + 255) / 256, rows, 8}, x, at::kByte);
    launch on(x);
    check(mi355x_mx4_quantize(type, x.const_data_ptr(), row_step(x), rows, k, (uint8_t *) codes.mutable_data_ptr(),
                              (uint8_t *) scales.mutable_data_ptr(), on.stream), "mx4_quantize");
    return {codes, scales};
}

Tensor dequantize(const Tensor & codes, const Tensor & scales, at::ScalarType dtype) {
    const mx4 m = check_mx4(codes, scales, "m", 2);
    const int type = elem_type(dtype, "dtype");
    Tensor y = fresh({m.rows, m.k}, codes, dtype);
    launch on(codes);
    check(mi355x_mx4_dequantize(bytes(codes), bytes(scales), m.rows, m.k, type, y.mutable_data_ptr(), on.stream), "mx4_dequantize");
    return y;
}

// the x of a product: float rows, or with x_scales MXFP4 rows
struct operand {
    int type;
    int64_t rows, step;
    const uint8_t * scales;
    at::ScalarType out;   // unless the caller asks for another
};

operand check_operand(const Tensor & x, const std::optional<Tensor> & x_scales, const Tensor & w, int64_t k) {
    beside(x, "x", w);
    operand o;
    int64_t have;
    if (x_scales) {
        const mx4 m = check_mx4(x, *x_scales, "x", 2);
        o = {MI355X_MX4, m.rows, m.k, bytes(*x_scales), at::kFloat};
        have = m.k;
    } else {
        const int type = matrix(x, "x");
        o = {type, x.size(0), row_step(x), nullptr, x.scalar_type()};
        have = x.size(1);
    }
    TORCH_CHECK_VALUE(have == k, "x: rows of ", k, " elements are wanted, got ", have);
    return o;
}

struct workspace {
    Tensor t;
    void * p = nullptr;
    int64_t size;
    workspace(int64_t size, const Tensor & like) : size(size) {
        if (size > 0) {
            t = fresh({size}, like, at::kByte);
            p = t.mutable_data_ptr();
        }
    }
};

Tensor mul_mat(const Tensor & w_codes, const Tensor & w_scales, const Tensor & x, const std::optional<Tensor> & x_scales,
               std::optional<at::ScalarType> dtype) {
    const mx4 w = check_mx4(w_codes, w_scales, "w", 2);
    const operand o = check_operand(x, x_scales, w_codes, w.k);
    const at::ScalarType out = dtype.value_or(o.out);
    const int ytype = elem_type(out, "dtype");
    Tensor y = fresh({o.rows, w.rows}, w_codes, out);
    const workspace work(mi355x_mx4_mul_mat_workspace(w.rows, w.k, o.type, o.rows), w_codes);
    launch on(w_codes);
    check(mi355x_mx4_mul_mat(bytes(w_codes), bytes(w_scales), w.rows, w.k, o.type, x.const_data_ptr(), o.scales, o.step, o.rows,
                             ytype, y.mutable_data_ptr(), work.p, work.size, on.stream), "mx4_mul_mat");
    return y;
}

Tensor mul_mat_id(const Tensor & w_codes, const Tensor & w_scales, const Tensor & x, const std::optional<Tensor> & x_scales,
                  const Tensor & order, const Tensor & rank, const Tensor & offsets, bool x_sorted,
                  std::optional<at::ScalarType> dtype) {
    const mx4 w = check_mx4(w_codes, w_scales, "w", 3);
    const plan p = check_plan(order, rank, offsets, w_codes);
    TORCH_CHECK_VALUE(w_codes.size(0) == p.experts, "w: ", w_codes.size(0), " experts, the plan has ", p.experts);
    const operand o = check_operand(x, x_scales, w_codes, w.k);
    TORCH_CHECK_VALUE(o.rows == (x_sorted ? p.t * p.used : p.t), "x: ", x_sorted ? p.t * p.used : p.t, " rows are wanted, got ",
                      o.rows);
    const at::ScalarType out = dtype.value_or(o.out);
    const int ytype = elem_type(out, "dtype");
    Tensor y = fresh({p.t * p.used, w.rows}, w_codes, out);
    const workspace work(mi355x_mx4_mul_mat_id_workspace(w.rows, w.k, p.experts, o.type, p.t, p.used, x_sorted), w_codes);
    launch on(w_codes);
    check(mi355x_mx4_mul_mat_id(bytes(w_codes), bytes(w_scales), w.rows, w.k, p.experts, o.type, x.const_data_ptr(), o.scales,
                                o.step, p.t, p.used, x_sorted, ints(order), ints(offsets), ytype, y.mutable_data_ptr(), work.p,
                                work.size, on.stream), "mx4_mul_mat_id");
    return y;
}

std::tuple<Tensor, Tensor, Tensor> sort(const Tensor & ids, int64_t n_expert) {
    on_gpu(ids, "ids");
    plain(ids, "ids");
    TORCH_CHECK_TYPE(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, "ids: int32 or int64 is wanted, got ",
                     ids.scalar_type());
    TORCH_CHECK_VALUE(ids.dim() == 2 && ids.is_contiguous(), "ids: a contiguous [T, used] tensor is wanted, got ", ids.sizes(),
                      ", strides ", ids.strides());
    const int64_t t = ids.size(0), used = ids.size(1);
    check_routing(used, n_expert);
    Tensor order = fresh({t * used}, ids, at::kInt), rank = fresh({t, used}, ids, at::kInt), offsets = fresh({n_expert + 1}, ids, at::kInt);
    const workspace work(mi355x_moe_sort_workspace(t, used, n_expert), ids);
    launch on(ids);
    check(mi355x_moe_sort(ids.const_data_ptr(), (int) ids.element_size(), t, used, n_expert, (int32_t *) order.mutable_data_ptr(),
                          (int32_t *) rank.mutable_data_ptr(), (int32_t *) offsets.mutable_data_ptr(),
                          work.p, work.size, on.stream), "moe_sort");
    return {order, rank, offsets};
}

Tensor gather(const Tensor & x, const Tensor & order, const Tensor & rank, const Tensor & offsets) {
    const int type = matrix(x, "x");
    const plan p = check_plan(order, rank, offsets, x);
    TORCH_CHECK_VALUE(x.size(0) == p.t, "x: ", x.size(0), " rows, the plan has ", p.t, " tokens");
    Tensor xs = fresh({p.t * p.used, x.size(1)}, x, x.scalar_type());
    launch on(x);
    check(mi355x_moe_gather(type, x.const_data_ptr(), row_step(x), p.t, x.size(1), p.used, ints(order), ints(rank),
                            xs.mutable_data_ptr(), on.stream), "moe_gather");
    return xs;
}

// rows in the plan's order: [T * used, D]
void check_sorted(const Tensor & ys, const plan & p) {
    TORCH_CHECK_VALUE(ys.size(0) == p.t * p.used, "ys: ", ys.size(0), " rows, the plan has ", p.t * p.used, " pairs");
}

Tensor combine(const Tensor & ys, const Tensor & order, const Tensor & rank, const Tensor & offsets,
               const std::optional<Tensor> & weights) {
    const int type = matrix(ys, "ys");
    const plan p = check_plan(order, rank, offsets, ys);
    check_sorted(ys, p);
    if (weights) {
        no_gradient(*weights, "weights");
        whole(*weights, "weights", ys, at::kFloat, {p.t, p.used});
    }
    Tensor y = fresh({p.t, ys.size(1)}, ys, ys.scalar_type());
    launch on(ys);
    check(mi355x_moe_combine(type, ys.const_data_ptr(), row_step(ys), p.t, ys.size(1), p.used, ints(rank),
                             weights ? (const float *) weights->const_data_ptr() : nullptr, y.mutable_data_ptr(), on.stream),
          "moe_combine");
    return y;
}

std::tuple<Tensor, Tensor> combine_back(const Tensor & dy, const Tensor & ys, const Tensor & order, const Tensor & rank,
                                        const Tensor & offsets, const Tensor & weights) {
    const int type = matrix(ys, "ys");
    const plan p = check_plan(order, rank, offsets, ys);
    check_sorted(ys, p);
    beside(dy, "dy", ys);
    matrix(dy, "dy");
    TORCH_CHECK_VALUE(dy.size(0) == p.t && dy.size(1) == ys.size(1), "dy: ", p.t, " rows of ", ys.size(1), " are wanted, got ", dy.sizes());
    TORCH_CHECK_TYPE(dy.scalar_type() == ys.scalar_type(), "dy: ", ys.scalar_type(), " is wanted, as ys has, got ", dy.scalar_type());
    no_gradient(weights, "weights");
    whole(weights, "weights", ys, at::kFloat, {p.t, p.used});
    Tensor dys = fresh({p.t * p.used, ys.size(1)}, ys, ys.scalar_type()), dw = fresh({p.t, p.used}, ys, at::kFloat);
    launch on(ys);
    check(mi355x_moe_combine_back(type, dy.const_data_ptr(), row_step(dy), ys.const_data_ptr(), row_step(ys), p.t, ys.size(1), p.used,
                                  ints(order), ints(rank), (const float *) weights.const_data_ptr(), dys.mutable_data_ptr(),
                                  (float *) dw.mutable_data_ptr(), on.stream), "moe_combine_back");
    return {dys, dw};
}

}  // namespace

PYBIND11_MODULE(_device_ops, m) {
    using free_gil = py::call_guard<py::gil_scoped_release>;
    m.def("quantize", &quantize, free_gil());
    m.def("dequantize", &dequantize, free_gil());
    m.def("mul_mat", &mul_mat, free_gil());
    m.def("mul_mat_id", &mul_mat_id, free_gil());
    m.def("sort", &sort, free_gil());
    m.def("gather", &gather, free_gil());
    m.def("combine", &combine, free_gil());
    m.def("combine_back", &combine_back, free_gil());
}
