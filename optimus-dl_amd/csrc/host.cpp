// The plain case of the Python wrappers in native.py, in C++: checks, output allocation and the call of the C entry.
//
// Every function takes what its wrapper takes and answers None where the call is not the plain one (a tensor that is not
// dense, aligned or of the expected type, an output of the caller's that does not fit): the wrapper then goes the long way,
// which copies or refuses.  An int is the status of a C entry that refused.  A step of a few hundred tokens waits for
// the host, and of its time a third went into the wrappers: per call 5 to 9 us of Python around 3.7 us of launch, here 1 to 2.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>
#include <torch/version.h>

#include <cstdint>

#include "../../include/odl_fp8.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using i64 = int64_t;

namespace {

constexpr i64 kParts = ODL_FP8_AMAX_PARTS;

// entries of the C library: their types from the header, their addresses from native.py, which has loaded it
decltype(&odl_fp8_amax_parts) amax_parts_c;
decltype(&odl_fp8_cast_dynamic_padded) cast_dynamic_c;
decltype(&odl_fp8_quantise_small) quantise_small_c;
decltype(&odl_fp8_gemm_swiglu) gemm_swiglu_c;
decltype(&odl_fp8_cast_delayed_padded) cast_delayed_c;
decltype(&odl_fp8_cast_delayed_many) cast_delayed_many_c;
decltype(&odl_fp8_amax_parts_colsum) amax_colsum_c;
decltype(&odl_fp8_amax_parts_slabs) amax_slabs_c;
decltype(&odl_fp8_slabs_colsum) slabs_colsum_c;
decltype(&odl_fp8_cast_dynamic_colsum) cast_colsum_c;
decltype(&odl_fp8_swiglu_amax_parts) swiglu_c;
decltype(&odl_fp8_swiglu_bwd_amax_parts) swiglu_bwd_c;
decltype(&odl_fp8_gelu_amax_parts) gelu_c;
decltype(&odl_fp8_gelu_bwd_amax_parts) gelu_bwd_c;
decltype(&odl_fp8_gelu_bwd_slabs) gelu_bwd_slabs_c;
decltype(&odl_fp8_rmsnorm_amax_parts) rmsnorm_c;
decltype(&odl_fp8_rmsnorm_bwd) rmsnorm_bwd_c;
decltype(&odl_fp8_layernorm_amax_parts) layernorm_c;
decltype(&odl_fp8_layernorm_bwd) layernorm_bwd_c;
decltype(&odl_fp8_amax_rowcol) amax_rowcol_c;
decltype(&odl_fp8_cast_rowcol_padded) cast_rowcol_c;
decltype(&odl_fp8_gemm_nt_hinted) gemm_nt_c;
decltype(&odl_fp8_gemm_group_route) group_route_c;
decltype(&odl_fp8_gemm_nt_group) gemm_nt_group_c;
decltype(&odl_fp8_gemm_chain_route) chain_route_c;
decltype(&odl_fp8_gemm_nt_chain) gemm_nt_chain_c;
decltype(&odl_fp8_gemm_layouts) gemm_layouts_c;
decltype(&odl_fp8_gemm_runs) runs_c;
decltype(&odl_fp8_mx_cast_padded) mx_cast_c;
decltype(&odl_fp8_block_cast) block_cast_c;
decltype(&odl_fp8_mx_gemm_nt_hinted) mx_gemm_nt_c;
decltype(&odl_fp8_last_error) last_error_c;
decltype(&odl_fp8_residual_norm) residual_norm_c;
decltype(&odl_fp8_residual_norm_bwd) residual_norm_bwd_c;
decltype(&odl_fp8_token_logprobs_workspace) logprobs_workspace_c;
decltype(&odl_fp8_token_logprobs) logprobs_c;
decltype(&odl_fp8_token_logprobs_bwd) logprobs_bwd_c;
decltype(&odl_fp8_fp4_linear_runs) fp4_runs_c;
decltype(&odl_fp8_fp4_linear) fp4_linear_c;

template <class F>
void take(F &f, const py::dict &d, const char *name) { f = reinterpret_cast<F>(py::cast<uintptr_t>(d[name])); }

void bind(const py::dict &d) {
    take(amax_parts_c, d, "odl_fp8_amax_parts");
    take(cast_dynamic_c, d, "odl_fp8_cast_dynamic_padded");
    take(quantise_small_c, d, "odl_fp8_quantise_small");
    take(gemm_swiglu_c, d, "odl_fp8_gemm_swiglu");
    take(cast_delayed_c, d, "odl_fp8_cast_delayed_padded");
    take(cast_delayed_many_c, d, "odl_fp8_cast_delayed_many");
    take(amax_colsum_c, d, "odl_fp8_amax_parts_colsum");
    take(amax_slabs_c, d, "odl_fp8_amax_parts_slabs");
    take(slabs_colsum_c, d, "odl_fp8_slabs_colsum");
    take(cast_colsum_c, d, "odl_fp8_cast_dynamic_colsum");
    take(swiglu_c, d, "odl_fp8_swiglu_amax_parts");
    take(swiglu_bwd_c, d, "odl_fp8_swiglu_bwd_amax_parts");
    take(gelu_c, d, "odl_fp8_gelu_amax_parts");
    take(gelu_bwd_c, d, "odl_fp8_gelu_bwd_amax_parts");
    take(gelu_bwd_slabs_c, d, "odl_fp8_gelu_bwd_slabs");
    take(rmsnorm_c, d, "odl_fp8_rmsnorm_amax_parts");
    take(rmsnorm_bwd_c, d, "odl_fp8_rmsnorm_bwd");
    take(layernorm_c, d, "odl_fp8_layernorm_amax_parts");
    take(layernorm_bwd_c, d, "odl_fp8_layernorm_bwd");
    take(amax_rowcol_c, d, "odl_fp8_amax_rowcol");
    take(cast_rowcol_c, d, "odl_fp8_cast_rowcol_padded");
    take(gemm_nt_c, d, "odl_fp8_gemm_nt_hinted");
    take(group_route_c, d, "odl_fp8_gemm_group_route");
    take(gemm_nt_group_c, d, "odl_fp8_gemm_nt_group");
    take(chain_route_c, d, "odl_fp8_gemm_chain_route");
    take(gemm_nt_chain_c, d, "odl_fp8_gemm_nt_chain");
    take(gemm_layouts_c, d, "odl_fp8_gemm_layouts");
    take(runs_c, d, "odl_fp8_gemm_runs");
    take(mx_cast_c, d, "odl_fp8_mx_cast_padded");
    take(block_cast_c, d, "odl_fp8_block_cast");
    take(mx_gemm_nt_c, d, "odl_fp8_mx_gemm_nt_hinted");
    take(last_error_c, d, "odl_fp8_last_error");
    take(residual_norm_c, d, "odl_fp8_residual_norm");
    take(residual_norm_bwd_c, d, "odl_fp8_residual_norm_bwd");
    take(logprobs_workspace_c, d, "odl_fp8_token_logprobs_workspace");
    take(logprobs_c, d, "odl_fp8_token_logprobs");
    take(logprobs_bwd_c, d, "odl_fp8_token_logprobs_bwd");
    take(fp4_runs_c, d, "odl_fp8_fp4_linear_runs");
    take(fp4_linear_c, d, "odl_fp8_fp4_linear");
}

// as ctypes does: other Python threads run while a launch waits for room in its queue
template <class F, class... A>
int call(F entry, A... args) {
    py::gil_scoped_release unlocked;
    return entry(args...);
}

// an address, as whatever pointer the entry takes
struct Address {
    void *p;
    template <class T>
    operator T *() const { return static_cast<T *>(p); }
};
Address ptr(const Tensor &t) { return {t.data_ptr()}; }
Address ptr(const OptTensor &t) { return {t ? t->data_ptr() : nullptr}; }
Address str(i64 stream) { return {reinterpret_cast<void *>(stream)}; }
bool aligned(const Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
int src_of(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kFloat ? 1 : -1; }
bool dense(const Tensor &t) { return t.is_cuda() && t.is_contiguous() && t.layout() == at::kStrided; }
bool source2d(const Tensor &t) { return dense(t) && t.dim() == 2 && src_of(t) >= 0; }
bool codes2d(const Tensor &t) { return dense(t) && t.dim() == 2 && t.scalar_type() == at::kByte; }
bool floats(const Tensor &t, i64 n) { return dense(t) && t.scalar_type() == at::kFloat && t.numel() == n; }
bool bf16(const Tensor &t) { return dense(t) && t.scalar_type() == at::kBFloat16 && aligned(t); }
Tensor bytes(const Tensor &like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kByte)); }
Tensor f32(const Tensor &like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kFloat)); }
py::object none() { return py::none(); }
py::object status(int rc) { return py::int_(rc); }
py::object obj(const OptTensor &t) { return t ? py::cast(*t) : py::none(); }

// an output of transposed codes: the caller's, if it fits, or a new one
bool transposed_out(const Tensor &x, const OptTensor &given, bool want, i64 cols, i64 rows, OptTensor &out) {
    if (given) {
        if (!codes2d(*given) || given->size(0) != cols || given->size(1) != rows || given->device() != x.device()) return false;
        out = given;
    } else if (want) out = bytes(x, {cols, rows});
    return true;
}

py::object amax_parts(const Tensor &x, i64 stream) {
    if (!source2d(x)) return none();
    Tensor parts = f32(x, {kParts});
    const int rc = call(amax_parts_c, ptr(x), src_of(x), x.size(0), x.size(1), ptr(parts), str(stream));
    return rc ? status(rc) : py::cast(parts);
}

py::object cast_dynamic(const Tensor &x, const Tensor &parts, int fmt, int margin, bool want_q, bool want_t, const OptTensor &out_t,
                        const std::optional<i64> &rows_out, i64 stream) {
    if (!source2d(x) || !(want_q || want_t || out_t)) return none();
    const i64 rows = x.size(0), cols = x.size(1), n = rows_out.value_or(rows);
    if (!floats(parts, kParts)) return none();
    OptTensor q, q_t;
    if (!transposed_out(x, out_t, want_t, cols, n, q_t)) return none();
    if (want_q) q = bytes(x, {n, cols});
    Tensor dyn = f32(x, {3, 1});
    const int rc = call(cast_dynamic_c, ptr(x), src_of(x), rows, cols, n, ptr(parts), fmt, margin, ptr(q), ptr(q_t), ptr(dyn), str(stream));
    if (rc) return status(rc);
    return py::make_tuple(obj(q), obj(q_t), dyn.select(0, 0), dyn.select(0, 1), dyn.select(0, 2));
}

// a small tensor in one launch, row-major codes only
py::object quantise_small(const Tensor &x, int fmt, int margin, i64 stream) {
    const i64 n = x.numel();
    if (!source2d(x) || n == 0 || n * x.element_size() > ODL_FP8_SMALL_BYTES || n % 16 || !aligned(x)) return none();
    Tensor q = bytes(x, {x.size(0), x.size(1)}), dyn = f32(x, {3, 1});
    const int rc = call(quantise_small_c, ptr(x), src_of(x), n, fmt, margin, ptr(q), ptr(dyn), str(stream));
    return rc ? status(rc) : py::make_tuple(q, py::none(), dyn.select(0, 0), dyn.select(0, 1), dyn.select(0, 2));
}

py::object gemm_swiglu(const Tensor &x, const Tensor &gate, const Tensor &up, int fx, int fw, const Tensor &sx, const Tensor &sg, const Tensor &su,
                       i64 stream) {
    if (!codes2d(x) || !codes2d(gate) || !codes2d(up) || gate.sizes() != up.sizes() || x.size(1) != gate.size(1) || !floats(sx, 1) || !floats(sg, 1) ||
        !floats(su, 1))
        return none();
    Tensor h = at::empty({x.size(0), gate.size(0)}, x.options().dtype(at::kBFloat16)), parts = f32(x, {kParts});
    const int rc = call(gemm_swiglu_c, ptr(x), ptr(gate), ptr(up), x.size(0), gate.size(0), x.size(1), fx, fw, ptr(sx), ptr(sg), ptr(su), ptr(h),
                        ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(h, parts);
}

py::object cast_delayed(const Tensor &x, const Tensor &scale, int fmt, const OptTensor &parts, bool want_q, bool want_t, const OptTensor &out_t,
                        const std::optional<i64> &rows_out, i64 stream) {
    if (!source2d(x) || !floats(scale, 1) || (parts && !floats(*parts, kParts)) || !(want_q || want_t || out_t)) return none();
    const i64 rows = x.size(0), cols = x.size(1), n = rows_out.value_or(rows);
    OptTensor q, q_t;
    if (!transposed_out(x, out_t, want_t, cols, n, q_t)) return none();
    if (want_q) q = bytes(x, {n, cols});
    Tensor inv = f32(x, {1});
    const int rc = call(cast_delayed_c, ptr(x), src_of(x), rows, cols, n, ptr(scale), fmt, ptr(q), ptr(q_t), ptr(parts), ptr(inv), str(stream));
    return rc ? status(rc) : py::make_tuple(obj(q), obj(q_t), inv);
}

py::object cast_delayed_many(const Tensor &x, const std::vector<Tensor> &scales, int fmt, const std::vector<Tensor> &parts, i64 rows_out, i64 stream) {
    const size_t n = scales.size();
    if (n < 1 || n > 4 || parts.size() != n || !source2d(x) || x.numel() == 0 || x.size(1) % 8 || rows_out % 16 || rows_out < x.size(0) || !aligned(x))
        return none();
    const float *s[4];
    float *p[4], *inv[4];
    uint8_t *q[4], *q_t[4];
    py::list made(n);
    Tensor invs = f32(x, {(i64)n});
    for (size_t i = 0; i < n; ++i) {
        if (!floats(scales[i], 1) || !floats(parts[i], kParts)) return none();
        Tensor a = bytes(x, {rows_out, x.size(1)}), b = bytes(x, {x.size(1), rows_out});
        s[i] = ptr(scales[i]), p[i] = ptr(parts[i]), inv[i] = static_cast<float *>(ptr(invs)) + i, q[i] = ptr(a), q_t[i] = ptr(b);
        made[i] = py::make_tuple(a, b, invs.narrow(0, (i64)i, 1));
    }
    const int rc = call(cast_delayed_many_c, ptr(x), src_of(x), x.size(0), x.size(1), rows_out, (int)n, s, fmt, q, q_t, p, inv, str(stream));
    return rc ? status(rc) : py::object(made);
}

py::object amax_colsum(const Tensor &x, bool finish, i64 stream) {
    if (!source2d(x)) return none();
    if (!finish && x.size(1) % 8 == 0 && aligned(x)) {
        Tensor parts = f32(x, {kParts}), ws = f32(x, {kParts, ODL_FP8_COLSUM_WORKSPACE / kParts});
        const int rc = call(amax_slabs_c, ptr(x), src_of(x), x.size(0), x.size(1), ptr(parts), ptr(ws), str(stream));
        return rc ? status(rc) : py::make_tuple(parts, ws);
    }
    Tensor parts = f32(x, {kParts}), sums = f32(x, {x.size(1)}), ws = f32(x, {ODL_FP8_COLSUM_WORKSPACE});
    const int rc = call(amax_colsum_c, ptr(x), src_of(x), x.size(0), x.size(1), ptr(parts), ptr(sums), ptr(ws), str(stream));
    return rc ? status(rc) : py::make_tuple(parts, sums);
}

// the column sums of x from the slabs that amax_colsum(x, false) or the producer of x left
py::object slabs_colsum(const Tensor &x, const Tensor &slabs, i64 stream) {
    if (!source2d(x) || x.numel() == 0 || !floats(slabs, ODL_FP8_COLSUM_WORKSPACE)) return none();
    Tensor sums = f32(x, {x.size(1)});
    const int rc = call(slabs_colsum_c, ptr(slabs), src_of(x), x.size(0), x.size(1), ptr(sums), str(stream));
    return rc ? status(rc) : py::cast(sums);
}

py::object cast_colsum(const Tensor &x, const Tensor &parts, const Tensor &slabs, int fmt, int margin, i64 rows_out, int odt, i64 stream) {
    if (!source2d(x) || !aligned(x) || !floats(parts, kParts) || !floats(slabs, ODL_FP8_COLSUM_WORKSPACE) || x.size(1) % 8) return none();
    const i64 rows = x.size(0), cols = x.size(1);
    Tensor q = bytes(x, {rows_out, cols}), q_t = bytes(x, {cols, rows_out}), dyn = f32(x, {3});
    Tensor sums = at::empty({cols}, x.options().dtype(odt ? at::kFloat : at::kBFloat16));
    const int rc = call(cast_colsum_c, ptr(x), src_of(x), rows, cols, rows_out, ptr(parts), fmt, margin, ptr(q), ptr(q_t), ptr(dyn), ptr(slabs), ptr(sums),
                        odt, str(stream));
    return rc ? status(rc) : py::make_tuple(q, q_t, dyn.narrow(0, 2, 1), sums);
}

i64 last(const Tensor &t) { return t.dim() ? t.size(-1) : 1; }

py::object swiglu(const Tensor &gate, const Tensor &up, i64 stream) {
    if (!bf16(gate) || !bf16(up) || gate.sizes() != up.sizes()) return none();
    const i64 cols = last(gate), rows = gate.numel() / std::max<i64>(cols, 1);
    Tensor h = at::empty_like(gate), parts = f32(gate, {kParts});
    const int rc = call(swiglu_c, ptr(gate), ptr(up), rows, cols, ptr(h), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(h, parts);
}

py::object swiglu_bwd(const Tensor &dh, const Tensor &gate, const Tensor &up, i64 stream) {
    if (!bf16(dh) || !bf16(gate) || !bf16(up) || gate.sizes() != up.sizes() || gate.sizes() != dh.sizes()) return none();
    const i64 cols = last(gate), rows = gate.numel() / std::max<i64>(cols, 1);
    Tensor dg = at::empty_like(gate), du = at::empty_like(up), parts = f32(gate, {2 * kParts});
    Tensor pg = parts.narrow(0, 0, kParts), pu = parts.narrow(0, kParts, kParts);
    const int rc = call(swiglu_bwd_c, ptr(dh), ptr(gate), ptr(up), rows, cols, ptr(dg), ptr(du), ptr(pg), ptr(pu), str(stream));
    return rc ? status(rc) : py::make_tuple(dg, du, pg, pu);
}

py::object gelu(const Tensor &x, const Tensor &table, i64 stream) {
    if (!bf16(x)) return none();
    const i64 cols = last(x), rows = x.numel() / std::max<i64>(cols, 1);
    Tensor y = at::empty_like(x), parts = f32(x, {kParts});
    const int rc = call(gelu_c, ptr(x), rows, cols, ptr(table), ptr(y), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(y, parts);
}

py::object gelu_bwd(const Tensor &dy, const Tensor &x, const Tensor &table, i64 stream) {
    if (!bf16(dy) || !bf16(x) || dy.sizes() != x.sizes()) return none();
    const i64 cols = last(x), rows = x.numel() / std::max<i64>(cols, 1);
    Tensor dx = at::empty_like(x), parts = f32(x, {kParts});
    const int rc = call(gelu_bwd_c, ptr(dy), ptr(x), rows, cols, ptr(table), ptr(dx), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(dx, parts);
}

py::object gelu_bwd_slabs(const Tensor &dy, const Tensor &x, const Tensor &table, i64 stream) {
    if (!bf16(dy) || !bf16(x) || dy.sizes() != x.sizes() || x.numel() == 0) return none();
    const i64 cols = last(x), rows = x.numel() / cols;
    if (cols % 8 || cols > kParts * 256) return none();
    Tensor dx = at::empty_like(x), parts = f32(x, {kParts}), ws = f32(x, {kParts, ODL_FP8_COLSUM_WORKSPACE / kParts});
    const int rc = call(gelu_bwd_slabs_c, ptr(dy), ptr(x), rows, cols, ptr(table), ptr(dx), ptr(parts), ptr(ws), str(stream));
    return rc ? status(rc) : py::make_tuple(dx, parts, ws);
}

// rows of a norm: dense, aligned, with vectors of the row length in fp32 on the same device
bool norm_input(const Tensor &x) { return dense(x) && src_of(x) >= 0 && x.dim() > 0 && aligned(x); }
bool norm_vector(const Tensor &w, const Tensor &x) { return floats(w, x.size(-1)) && aligned(w) && w.device() == x.device(); }

py::object rmsnorm(const Tensor &x, const Tensor &w, double eps, i64 stream) {
    if (!norm_input(x) || !norm_vector(w, x)) return none();
    const i64 cols = x.size(-1), rows = x.numel() / std::max<i64>(cols, 1);
    Tensor y = at::empty(x.sizes(), x.options().dtype(at::kBFloat16)), rstd = f32(x, x.sizes().slice(0, x.dim() - 1)), parts = f32(x, {kParts});
    const int rc = call(rmsnorm_c, ptr(x), src_of(x), ptr(w), rows, cols, (float)eps, ptr(y), ptr(rstd), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(y, rstd, parts);
}

py::object rmsnorm_bwd(const Tensor &dy, const Tensor &x, const Tensor &w, const Tensor &rstd, i64 stream) {
    if (!bf16(dy) || !norm_input(x) || dy.sizes() != x.sizes() || !norm_vector(w, x)) return none();
    const i64 cols = x.size(-1), rows = x.numel() / std::max<i64>(cols, 1);
    if (!floats(rstd, rows)) return none();
    Tensor dx = at::empty_like(x), dw = f32(x, {cols}), ws = f32(x, {ODL_FP8_RMSNORM_BWD_SLABS * cols});
    const int rc = call(rmsnorm_bwd_c, ptr(dy), ptr(x), src_of(x), ptr(w), ptr(rstd), rows, cols, ptr(dx), ptr(dw), ptr(ws), str(stream));
    return rc ? status(rc) : py::make_tuple(dx, dw);
}

py::object layernorm(const Tensor &x, const Tensor &w, const OptTensor &b, double eps, i64 stream) {
    if (!norm_input(x) || !norm_vector(w, x) || (b && !norm_vector(*b, x))) return none();
    const i64 cols = x.size(-1), rows = x.numel() / std::max<i64>(cols, 1);
    std::vector<i64> lead{2};
    for (int d = 0; d + 1 < x.dim(); ++d) lead.push_back(x.size(d));
    Tensor y = at::empty(x.sizes(), x.options().dtype(at::kBFloat16)), stats = f32(x, lead), parts = f32(x, {kParts});
    Tensor mean = stats.select(0, 0), rstd = stats.select(0, 1);
    const int rc = call(layernorm_c, ptr(x), src_of(x), ptr(w), ptr(b), rows, cols, (float)eps, ptr(y), ptr(mean), ptr(rstd), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(y, mean, rstd, parts);
}

py::object layernorm_bwd(const Tensor &dy, const Tensor &x, const Tensor &w, const Tensor &mean, const Tensor &rstd, i64 stream) {
    if (!bf16(dy) || !norm_input(x) || dy.sizes() != x.sizes() || !norm_vector(w, x)) return none();
    const i64 cols = x.size(-1), rows = x.numel() / std::max<i64>(cols, 1);
    if (!floats(mean, rows) || !floats(rstd, rows)) return none();
    Tensor dx = at::empty_like(x), dwb = f32(x, {2 * cols}), ws = f32(x, {2 * ODL_FP8_RMSNORM_BWD_SLABS * cols});
    Tensor dw = dwb.narrow(0, 0, cols), db = dwb.narrow(0, cols, cols);
    const int rc = call(layernorm_bwd_c, ptr(dy), ptr(x), src_of(x), ptr(w), ptr(mean), ptr(rstd), rows, cols, ptr(dx), ptr(dw), ptr(db), ptr(ws),
                                   str(stream));
    return rc ? status(rc) : py::make_tuple(dx, dw, db);
}

py::object quantize_rowcol(const Tensor &x, int fmt, int margin, const std::optional<i64> &rows_out, i64 stream) {
    if (!source2d(x)) return none();
    const i64 rows = x.size(0), cols = x.size(1), n = rows_out.value_or(rows);
    const i64 pr = (rows + 3) / 4 * 4, pc = (cols + 3) / 4 * 4, o = pr + pc;      // every vector starts on a 16-byte boundary
    Tensor buf = f32(x, {3 * o});
    Tensor a_row = buf.narrow(0, 0, rows), a_col = buf.narrow(0, pr, cols), i_row = buf.narrow(0, 2 * o, rows), i_col = buf.narrow(0, 2 * o + pr, cols);
    float *base = buf.data_ptr<float>();
    Tensor q = bytes(x, {n, cols}), q_t = bytes(x, {cols, n});
    int rc = call(amax_rowcol_c, ptr(x), src_of(x), rows, cols, base, base + pr, str(stream));
    if (!rc)
        rc = call(cast_rowcol_c, ptr(x), src_of(x), rows, cols, n, base, base + pr, fmt, margin, ptr(q), ptr(q_t), base + o, base + 2 * o, base + o + pr,
                           base + 2 * o + pr, str(stream));
    return rc ? status(rc) : py::make_tuple(q, i_row, q_t, i_col, a_row, a_col);
}

bool out_fits(const OptTensor &out, i64 M, i64 N) { return !out || (dense(*out) && src_of(*out) >= 0 && out->dim() == 2 && out->size(0) == M && out->size(1) == N); }
Tensor result(const OptTensor &out, const Tensor &like, i64 M, i64 N, int odt) {
    return out ? *out : at::empty({M, N}, like.options().dtype(odt ? at::kFloat : at::kBFloat16));
}
bool small(i64 M, i64 N, i64 K) { return (M + 256) * K < (i64)1 << 31 && (N + 256) * K < (i64)1 << 31; }

// odt: 0 = bf16, 1 = fp32 (where no `out` decides).  split: K may be cut into runs, which the long way does.
py::object gemm_nt(const Tensor &a, const Tensor &b, int fa, int fb, const Tensor &sa, const Tensor &sb, const OptTensor &bias, int odt,
                   const OptTensor &out, bool accumulate, bool fresh, bool split, i64 stream) {
    if (!codes2d(a) || !codes2d(b) || a.size(1) != b.size(1)) return none();
    const i64 M = a.size(0), K = a.size(1), N = b.size(0), na = sa.numel(), nb = sb.numel();
    if ((na != 1 && na != M) || (nb != 1 && nb != N) || !floats(sa, na) || !floats(sb, nb) || (bias && !floats(*bias, N)) || !out_fits(out, M, N) ||
        (accumulate && !out) || (na > 1 && !aligned(sa)) || (nb > 1 && !aligned(sb)) || (bias && !aligned(*bias)))
        return none();
    if (split && small(M, N, K) && runs_c(M, N, K, 0) > 1) return none();
    Tensor c = result(out, a, M, N, odt);
    const int rc = call(gemm_nt_c, ptr(a), ptr(b), M, N, K, fa, fb, ptr(sa), na, ptr(sb), nb, ptr(bias), 1, ptr(c), src_of(c), accumulate, fresh, str(stream));
    return rc ? status(rc) : py::cast(c);
}

bool group_in_one_launch(const std::vector<i64> &M, const std::vector<i64> &N, i64 K, int odt) {
    return M.size() == N.size() && M.size() <= 4 && group_route_c((int)M.size(), M.data(), N.data(), K, odt) >= 0;
}

// Several products in one launch; None where they run one by one (each then in the way that is its own)
py::object gemm_nt_group(const std::vector<Tensor> &a, const std::vector<Tensor> &b, int fa, int fb, const std::vector<Tensor> &sa,
                         const std::vector<Tensor> &sb, int odt, bool fresh, i64 stream) {
    const size_t n = a.size();
    if (n < 2 || n > 4 || b.size() != n || sa.size() != n || sb.size() != n) return none();
    const uint8_t *pa[4], *pb[4];
    const float *psa[4], *psb[4];
    void *pc[4];
    i64 M[4], N[4];
    for (size_t s = 0; s < n; ++s) {
        if (!codes2d(a[s]) || !codes2d(b[s]) || a[s].size(1) != a[0].size(1) || b[s].size(1) != a[0].size(1) || !floats(sa[s], 1) || !floats(sb[s], 1) ||
            !aligned(a[s]) || !aligned(b[s]))
            return none();
        M[s] = a[s].size(0); N[s] = b[s].size(0);
        pa[s] = ptr(a[s]); pb[s] = ptr(b[s]); psa[s] = ptr(sa[s]); psb[s] = ptr(sb[s]);
    }
    const i64 K = a[0].size(1);
    if (group_route_c((int)n, M, N, K, odt) < 0) return none();
    py::list out;
    for (size_t s = 0; s < n; ++s) {
        Tensor c = result(OptTensor(), a[s], M[s], N[s], odt);
        pc[s] = ptr(c);
        out.append(c);
    }
    const int rc = call(gemm_nt_group_c, (int)n, pa, pb, M, N, K, fa, fb, psa, psb, pc, odt, fresh, str(stream));
    return rc ? status(rc) : py::object(out);
}

bool chain_in_one_launch(const std::vector<i64> &K, i64 M, i64 N) { return K.size() <= 4 && chain_route_c((int)K.size(), K.data(), M, N) >= 0; }

// The bf16 sum of several products in one launch
py::object gemm_nt_chain(const std::vector<Tensor> &a, const std::vector<Tensor> &b, int fa, int fb, const std::vector<Tensor> &sa,
                         const std::vector<Tensor> &sb, i64 stream) {
    const size_t n = a.size();
    if (n < 2 || n > 4 || b.size() != n || sa.size() != n || sb.size() != n) return none();
    const uint8_t *pa[4], *pb[4];
    const float *psa[4], *psb[4];
    i64 K[4];
    for (size_t s = 0; s < n; ++s) {
        if (!codes2d(a[s]) || !codes2d(b[s]) || a[s].size(0) != a[0].size(0) || b[s].size(0) != b[0].size(0) || a[s].size(1) != b[s].size(1)) return none();
        if (!floats(sa[s], 1) || !floats(sb[s], 1)) return none();
        K[s] = a[s].size(1);
        pa[s] = ptr(a[s]); pb[s] = ptr(b[s]); psa[s] = ptr(sa[s]); psb[s] = ptr(sb[s]);
    }
    Tensor c = result(OptTensor(), a[0], a[0].size(0), b[0].size(0), 0);
    const int rc = call(gemm_nt_chain_c, (int)n, pa, pb, K, a[0].size(0), b[0].size(0), fa, fb, psa, psb, ptr(c), str(stream));
    return rc ? status(rc) : py::cast(c);
}

// Not accumulating; whole tiles of the kernel that reads K-slow operands (the caller has checked: gemm_layouts_supported)
py::object gemm_layouts(const Tensor &a, const Tensor &b, int fa, int fb, bool a_slow, bool b_slow, const Tensor &sa, const Tensor &sb,
                        const OptTensor &out, int odt, bool split, i64 stream) {
    if (!codes2d(a) || !codes2d(b) || !floats(sa, 1) || !floats(sb, 1)) return none();
    const i64 M = a.size(a_slow ? 1 : 0), K = a.size(a_slow ? 0 : 1), N = b.size(b_slow ? 1 : 0);
    if (K != b.size(b_slow ? 0 : 1) || !out_fits(out, M, N) || M <= 0 || N <= 0 || M % 256 || N % 256 || K % 128 || K < 512 || !small(M, N, K)) return none();
    if (N * (i64)4 * 264 >= (i64)1 << 31 || (split && runs_c(M, N, K, a_slow || b_slow) > 1)) return none();
    Tensor c = result(out, a, M, N, odt);
    const int rc = call(gemm_layouts_c, ptr(a), ptr(b), M, N, K, fa, fb, a_slow, b_slow, ptr(sa), ptr(sb), ptr(c), src_of(c), str(stream));
    return rc ? status(rc) : py::cast(c);
}

// scale bytes of `rows` rows blocked along `length` elements, in the layout the streaming GEMM reads where the length allows
Tensor mx_scales(const Tensor &x, i64 rows, i64 length, int &layout) {
    layout = length % 128 == 0 && length > 0;
    return layout ? bytes(x, {length / 128, rows, 4}) : bytes(x, {rows, length / 32});
}

py::object mx_cast(const Tensor &x, int fmt, bool want_q, bool want_t, int rule, const std::optional<i64> &rows_out, i64 stream) {
    if (!source2d(x) || !(want_q || want_t)) return none();
    const i64 rows = x.size(0), cols = x.size(1), n = rows_out.value_or(rows);
    OptTensor q, s, q_t, s_t;
    int lay = 0, lay_t = 0;
    if (want_q) { q = bytes(x, {rows, cols}); s = mx_scales(x, rows, cols, lay); }
    if (want_t) { q_t = bytes(x, {cols, n}); s_t = mx_scales(x, cols, n, lay_t); }
    const int rc = call(mx_cast_c, ptr(x), src_of(x), rows, cols, n, fmt, ptr(q), ptr(s), lay, ptr(q_t), ptr(s_t), lay_t, rule, str(stream));
    return rc ? status(rc) : py::make_tuple(obj(q), obj(s), obj(q_t), obj(s_t));
}

py::object block_cast(const Tensor &x, int fmt, int margin, bool two_d, bool want_q, bool want_t, i64 stream) {
    if (!source2d(x) || !(want_q || want_t) || x.size(0) % 128 || x.size(1) % 128) return none();
    const i64 rows = x.size(0), cols = x.size(1);
    OptTensor q, s, q_t, s_t;
    if (want_q) { q = bytes(x, {rows, cols}); s = bytes(x, {cols / 128, rows, 4}); }
    if (want_t) { q_t = bytes(x, {cols, rows}); s_t = bytes(x, {rows / 128, cols, 4}); }
    const int rc = call(block_cast_c, ptr(x), src_of(x), rows, cols, fmt, margin, two_d, ptr(q), ptr(s), ptr(q_t), ptr(s_t), str(stream));
    return rc ? status(rc) : py::make_tuple(obj(q), obj(s), obj(q_t), obj(s_t));
}

py::object mx_gemm_nt(const Tensor &a, const Tensor &sa, const Tensor &b, const Tensor &sb, int fa, int fb, const OptTensor &bias, int odt,
                      const OptTensor &out, bool accumulate, bool fresh, bool split, i64 stream) {
    if (!codes2d(a) || !codes2d(b) || a.size(1) != b.size(1) || !dense(sa) || !dense(sb) || sa.scalar_type() != at::kByte || sb.scalar_type() != at::kByte)
        return none();
    const i64 M = a.size(0), K = a.size(1), N = b.size(0);
    // K-step-major scales only: what the casts of this package make wherever K has whole steps
    if (K % 128 || sa.dim() != 3 || sb.dim() != 3 || sa.size(0) != K / 128 || sa.size(1) != M || sa.size(2) != 4 || sb.size(0) != K / 128 ||
        sb.size(1) != N || sb.size(2) != 4)
        return none();
    if ((bias && !floats(*bias, N)) || !out_fits(out, M, N) || (accumulate && !out)) return none();
    if (split && small(M, N, K) && runs_c(M, N, K, 0) > 1) return none();
    Tensor c = result(out, a, M, N, odt);
    const int rc = call(mx_gemm_nt_c, ptr(a), ptr(sa), ptr(b), ptr(sb), 1, M, N, K, fa, fb, ptr(bias), ptr(c), src_of(c), accumulate, fresh, str(stream));
    return rc ? status(rc) : py::cast(c);
}

// the operands that both directions of the residual stream's step share
bool residual_operands(const Tensor &x, const Tensor &h, const Tensor &w, const OptTensor &post, const OptTensor &gate) {
    if (!norm_input(x) || !norm_input(h) || x.sizes() != h.sizes() || x.device() != h.device() || src_of(h) > src_of(x) || !norm_vector(w, x)) return false;
    if (x.size(-1) % 8 || x.size(-1) < 8 || x.size(-1) > 8192) return false;
    if (post && !norm_vector(*post, x)) return false;
    return !gate || (gate->device() == x.device() && (floats(*gate, 1) || floats(*gate, x.size(-1))));
}

py::object residual_norm(const Tensor &x, const Tensor &h, const Tensor &w, const OptTensor &post, const OptTensor &gate, double scale, double eps,
                         double post_eps, bool keep, i64 stream) {
    if (!residual_operands(x, h, w, post, gate)) return none();
    const i64 cols = x.size(-1), rows = x.numel() / cols;
    Tensor y = at::empty_like(x), z = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
    OptTensor stats, parts;
    if (keep) {
        stats = f32(x, {2, rows});
        parts = f32(x, {kParts});
    }
    const int rc = call(residual_norm_c, ptr(x), src_of(x), ptr(h), src_of(h), ptr(w), ptr(post), ptr(gate), gate ? gate->numel() : 0, rows, cols,
                        (float)scale, (float)eps, (float)post_eps, ptr(y), ptr(z), ptr(stats), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(y, z, obj(stats), obj(parts));
}

py::object residual_norm_bwd(const OptTensor &dy, const OptTensor &dz, const Tensor &x, const Tensor &h, const Tensor &w, const OptTensor &post,
                             const OptTensor &gate, double scale, const Tensor &stats, bool weights, i64 stream) {
    if (!residual_operands(x, h, w, post, gate)) return none();
    if (dy && (!norm_input(*dy) || dy->sizes() != x.sizes() || dy->scalar_type() != x.scalar_type() || dy->device() != x.device())) return none();
    if (dz && (!bf16(*dz) || dz->sizes() != x.sizes() || dz->device() != x.device())) return none();
    const i64 cols = x.size(-1), rows = x.numel() / cols, g = gate ? gate->numel() : 0;
    if (!floats(stats, 2 * rows) || stats.device() != x.device()) return none();
    Tensor dx = at::empty_like(x), dh = at::empty_like(h), parts = f32(x, {kParts});
    OptTensor dw, dpost, dgate, ws;
    if (weights) {
        dw = f32(x, {cols});
        if (post) dpost = f32(x, {cols});
        if (gate) dgate = f32(x, {g});
        ws = f32(x, {ODL_FP8_RESIDUAL_NORM_SLABS * (2 * cols + 1)});
    }
    const int rc = call(residual_norm_bwd_c, ptr(dy), ptr(dz), ptr(x), src_of(x), ptr(h), src_of(h), ptr(w), ptr(post), ptr(gate), g, rows, cols,
                        (float)scale, ptr(stats), ptr(dx), ptr(dh), ptr(parts), ptr(dw), ptr(dpost), ptr(dgate), ptr(ws), str(stream));
    return rc ? status(rc) : py::make_tuple(dx, dh, parts, obj(dw), obj(dpost), obj(dgate));
}

// logits [rows, columns], rows at any distance; their other form, of any shape, goes the long way
bool logits2d(const Tensor &l) { return l.is_cuda() && l.layout() == at::kStrided && l.dim() == 2 && src_of(l) >= 0 && l.numel() > 0 && l.stride(1) == 1 && l.stride(0) >= 0; }

py::object token_logprobs(const Tensor &l, const Tensor &targets, i64 vocab, int top_k, double inv_t, i64 ignore, bool keep, i64 stream) {
    if (!logits2d(l) || !dense(targets) || targets.scalar_type() != at::kLong || targets.numel() != l.size(0) || targets.device() != l.device()) return none();
    const i64 rows = l.size(0);
    if (vocab < 1 || vocab > l.size(1) || top_k < 0 || top_k > ODL_FP8_LOGPROBS_MAX_TOP) return none();
    Tensor out = f32(l, {2, rows});
    OptTensor stats, top, ids;
    if (keep) stats = f32(l, {2, rows});
    if (top_k) {
        top = f32(l, {rows, top_k});
        ids = at::empty({rows, top_k}, l.options().dtype(at::kLong));
    }
    const i64 need = logprobs_workspace_c(rows, vocab, top_k);
    OptTensor ws;
    if (need) ws = f32(l, {need});
    Tensor lp = out.select(0, 0), entropy = out.select(0, 1);
    const int rc = call(logprobs_c, ptr(l), src_of(l), rows, l.stride(0), vocab, targets.data_ptr<i64>(), ignore, (float)inv_t, top_k, ptr(lp), ptr(entropy),
                        ptr(stats), ptr(top), ptr(ids), ptr(ws), 4 * need, str(stream));
    return rc ? status(rc) : py::make_tuple(lp, entropy, obj(stats), obj(top), obj(ids));
}

bool row_gradient(const OptTensor &g, i64 n) { return !g || floats(*g, n); }

py::object token_logprobs_bwd(const Tensor &l, const Tensor &targets, i64 vocab, int top_k, double inv_t, i64 ignore, const OptTensor &ids,
                              const Tensor &stats, const Tensor &entropy, const OptTensor &dlp, const OptTensor &dent, const OptTensor &dtop, i64 stream) {
    if (!logits2d(l) || !dense(targets) || targets.scalar_type() != at::kLong || targets.numel() != l.size(0)) return none();
    const i64 rows = l.size(0), cols = l.size(1);
    if (!floats(stats, 2 * rows) || !floats(entropy, rows) || !row_gradient(dlp, rows) || !row_gradient(dent, rows) || !row_gradient(dtop, rows * top_k))
        return none();
    if (dtop && (!ids || !dense(*ids) || ids->scalar_type() != at::kLong || ids->numel() != rows * top_k)) return none();
    Tensor dl = at::empty({rows, cols}, l.options()), parts = f32(l, {kParts});
    const int rc = call(logprobs_bwd_c, ptr(l), src_of(l), rows, l.stride(0), vocab, cols, targets.data_ptr<i64>(), ignore, (float)inv_t, top_k, ptr(ids),
                        ptr(stats), ptr(entropy), ptr(dlp), ptr(dent), ptr(dtop), ptr(dl), ptr(parts), str(stream));
    return rc ? status(rc) : py::make_tuple(dl, parts);
}

py::object fp4_linear(const Tensor &x, const Tensor &codes, const Tensor &scales, const OptTensor &bias, i64 stream) {
    if (!x.is_cuda() || x.dim() != 2 || x.scalar_type() != at::kBFloat16 || x.stride(1) != 1 || x.stride(0) % 8 || !aligned(x) || !codes2d(codes) || !aligned(codes))
        return none();
    const i64 M = x.size(0), K = x.size(1), N = codes.size(0);
    if (x.stride(0) < K || x.stride(0) > (1 << 24) || codes.size(1) * 2 != K || !dense(scales) || scales.scalar_type() != at::kBFloat16 || scales.dim() != 2 || scales.size(0) != N || scales.size(1) < 1 ||
        K % scales.size(1) || codes.device() != x.device() || scales.device() != x.device())
        return none();
    if (bias && (!dense(*bias) || src_of(*bias) < 0 || bias->numel() != N || bias->device() != x.device())) return none();
    const int group = (int)(K / scales.size(1));
    const i64 partial = (i64)fp4_runs_c(M, N, K, group) * M * N;
    Tensor y = at::empty({M, N}, x.options());
    OptTensor ws;
    if (partial) ws = f32(x, {partial});
    const int rc = call(fp4_linear_c, ptr(x), x.stride(0), ptr(codes), ptr(scales), group, ptr(bias), bias ? src_of(*bias) : 0, M, N, K, ptr(y), ptr(ws), 4 * partial,
                        str(stream));
    return rc ? status(rc) : py::cast(y);
}

// ---- The same two as autograd nodes, for graphs without a recipe (which would be handed maxima, in Python).  Python's part of a
// node is 60 to 100 us of a step that computes for 20; these take 25.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// an entry's answer where no Python is on the way (the thread of a backward does not hold its lock)
void done(int rc, const char *what) {
    if (rc) throw std::runtime_error(std::string(what) + " refused: " + last_error_c());
}
OptTensor given(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
// dense and aligned, as the kernels read it
OptTensor dense_gradient(const Tensor &t) {
    if (!t.defined()) return {};
    Tensor d = t.contiguous();
    return aligned(d) ? d : d.clone(at::MemoryFormat::Contiguous);
}
// Gradients of kernels that autograd cannot see into: where a graph of the backward is recorded, what would differentiate them raises.
variable_list once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor &g : grads)
        if (g.defined()) {
            variable_list in{g.detach().set_requires_grad(true)};
            g = (*std::make_shared<torch::autograd::DelayedError>(std::string(what) + " can be differentiated once only", 1))(std::move(in))[0];
        }
    return grads;
}

struct ResidualNormNode : torch::autograd::Function<ResidualNormNode> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &h, const Tensor &w, const OptTensor &post, const OptTensor &gate, double scale,
                                 double eps, double post_eps, i64 stream) {
        const i64 cols = x.size(-1), rows = x.numel() / cols;
        Tensor y = at::empty_like(x), z = at::empty(x.sizes(), x.options().dtype(at::kBFloat16)), stats = f32(x, {2, rows});
        done(residual_norm_c(ptr(x), src_of(x), ptr(h), src_of(h), ptr(w), ptr(post), ptr(gate), gate ? gate->numel() : 0, rows, cols, (float)scale, (float)eps,
                             (float)post_eps, ptr(y), ptr(z), static_cast<float *>(ptr(stats)), nullptr, str(stream)),
             "odl_fp8_residual_norm");
        ctx->save_for_backward({x, h, w, post.value_or(Tensor()), gate.value_or(Tensor()), stats});
        ctx->set_materialize_grads(false);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["stream"] = stream;
        return {y, z};
    }

    static variable_list backward(AutogradContext *ctx, variable_list out) {
        variable_list grads(9);
        if (!out[0].defined() && !out[1].defined()) return grads;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &h = saved[1], &w = saved[2], &stats = saved[5];
        const OptTensor post = given(saved[3]), gate = given(saved[4]), dy = dense_gradient(out[0]), dz = dense_gradient(out[1]);
        {
            at::NoGradGuard quiet;
            const i64 cols = x.size(-1), rows = x.numel() / cols, g = gate ? gate->numel() : 0;
            const bool weights = ctx->needs_input_grad(2) || (post && ctx->needs_input_grad(3)) || (gate && ctx->needs_input_grad(post ? 4 : 3));
            Tensor dx = at::empty_like(x), dh = at::empty_like(h);
            OptTensor dw, dpost, dgate, ws;
            if (weights) {
                dw = f32(x, w.sizes());
                if (post) dpost = f32(x, post->sizes());
                if (gate) dgate = f32(x, gate->sizes());
                ws = f32(x, {ODL_FP8_RESIDUAL_NORM_SLABS * (2 * cols + 1)});
            }
            // (a node runs on the stream that its forward ran on)
            done(residual_norm_bwd_c(ptr(dy), ptr(dz), ptr(x), src_of(x), ptr(h), src_of(h), ptr(w), ptr(post), ptr(gate), g, rows, cols,
                                     (float)ctx->saved_data["scale"].toDouble(), ptr(stats), ptr(dx), ptr(dh), nullptr, ptr(dw), ptr(dpost), ptr(dgate), ptr(ws),
                                     str(ctx->saved_data["stream"].toInt())),
                 "odl_fp8_residual_norm_bwd");
            grads[0] = dx;
            grads[1] = dh;
            if (dw) grads[2] = *dw;
            if (dpost) grads[3] = *dpost;
            if (dgate) grads[4] = *dgate;
        }
        return once(std::move(grads), "residual_norm");
    }
};

py::object residual_norm_node(const Tensor &x, const Tensor &h, const Tensor &w, const OptTensor &post, const OptTensor &gate, double scale, double eps,
                              double post_eps, i64 stream) {
    if (!residual_operands(x, h, w, post, gate) || x.numel() == 0) return none();
    variable_list out;
    {
        py::gil_scoped_release unlocked;
        out = ResidualNormNode::apply(x, h, w, post, gate, scale, eps, post_eps, stream);
    }
    return py::make_tuple(out[0], out[1]);
}

struct TokenLogprobsNode : torch::autograd::Function<TokenLogprobsNode> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &targets, i64 vocab, i64 top_k, double inv_t, i64 ignore, i64 stream) {
        const Tensor l = logits.reshape({-1, logits.size(-1)});
        const i64 rows = l.size(0);
        const auto lead = logits.sizes().slice(0, logits.dim() - 1);
        Tensor lp = f32(l, lead), entropy = f32(l, lead), stats = f32(l, {2, rows}), top, ids;
        if (top_k) {
            std::vector<i64> shape(lead.begin(), lead.end());
            shape.push_back(top_k);
            top = f32(l, shape);
            ids = at::empty(shape, l.options().dtype(at::kLong));
        }
        const i64 need = logprobs_workspace_c(rows, vocab, (int)top_k);
        OptTensor ws;
        if (need) ws = f32(l, {need});
        done(logprobs_c(ptr(l), src_of(l), rows, l.stride(0), vocab, targets.data_ptr<i64>(), ignore, (float)inv_t, (int)top_k, ptr(lp), ptr(entropy), ptr(stats),
                        ptr(given(top)), ptr(given(ids)), ptr(ws), 4 * need, str(stream)),
             "odl_fp8_token_logprobs");
        ctx->save_for_backward({logits, targets, entropy, stats, ids});
        ctx->set_materialize_grads(false);
        ctx->saved_data["vocab"] = vocab;
        ctx->saved_data["top_k"] = top_k;
        ctx->saved_data["inv_t"] = inv_t;
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["stream"] = stream;
        if (!top_k) return {lp, entropy};
        ctx->mark_non_differentiable({ids});
        return {lp, entropy, top, ids};
    }

    static variable_list backward(AutogradContext *ctx, variable_list out) {
        variable_list grads(7);
        const i64 top_k = ctx->saved_data["top_k"].toInt();
        const bool tops = top_k && out[2].defined();
        if (!out[0].defined() && !out[1].defined() && !tops) return grads;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &targets = saved[1], &entropy = saved[2], &stats = saved[3];
        const OptTensor dlp = dense_gradient(out[0]), dent = dense_gradient(out[1]), dtop = tops ? dense_gradient(out[2]) : OptTensor(), ids = given(saved[4]);
        {
            at::NoGradGuard quiet;
            const Tensor l = logits.reshape({-1, logits.size(-1)});
            const i64 rows = l.size(0), cols = l.size(1);
            Tensor dl = at::empty({rows, cols}, l.options());
            done(logprobs_bwd_c(ptr(l), src_of(l), rows, l.stride(0), ctx->saved_data["vocab"].toInt(), cols, targets.data_ptr<i64>(), ctx->saved_data["ignore"].toInt(),
                                (float)ctx->saved_data["inv_t"].toDouble(), (int)top_k, ptr(ids), ptr(stats), ptr(entropy), ptr(dlp), ptr(dent), ptr(dtop), ptr(dl), nullptr,
                                str(ctx->saved_data["stream"].toInt())),
                 "odl_fp8_token_logprobs_bwd");
            grads[0] = dl.view(logits.sizes());
        }
        return once(std::move(grads), "token_logprobs");
    }
};

py::object token_logprobs_node(const Tensor &logits, const Tensor &targets, i64 vocab, i64 top_k, double inv_t, i64 ignore, i64 stream) {
    if (logits.dim() < 1 || logits.numel() == 0 || !dense(targets) || targets.scalar_type() != at::kLong || targets.device() != logits.device()) return none();
    if (!(logits.dim() == 2 ? logits2d(logits) : dense(logits) && src_of(logits) >= 0)) return none();
    if (vocab < 1 || vocab > logits.size(-1) || top_k < 0 || top_k > ODL_FP8_LOGPROBS_MAX_TOP || top_k > vocab) return none();
    // (what either direction of the kernels refuses is refused in front of the forward, by the wrapper)
    if (logits.size(-1) > 1 << 24 || logits.numel() / logits.size(-1) >= 1 << 22) return none();
    variable_list out;
    {
        py::gil_scoped_release unlocked;
        out = TokenLogprobsNode::apply(logits, targets, vocab, top_k, inv_t, ignore, stream);
    }
    if (!top_k) return py::make_tuple(out[0], out[1], py::none(), py::none());
    return py::make_tuple(out[0], out[1], out[2], out[3]);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.attr("abi_version") = ODL_FP8_ABI_VERSION;        // of the header this was compiled with
    m.attr("torch_version") = TORCH_VERSION;
    m.def("bind", &bind);
    m.def("amax_parts", &amax_parts);
    m.def("cast_dynamic", &cast_dynamic);
    m.def("quantise_small", &quantise_small);
    m.def("gemm_swiglu", &gemm_swiglu);
    m.def("cast_delayed", &cast_delayed);
    m.def("cast_delayed_many", &cast_delayed_many);
    m.def("amax_colsum", &amax_colsum);
    m.def("slabs_colsum", &slabs_colsum);
    m.def("cast_colsum", &cast_colsum);
    m.def("swiglu", &swiglu);
    m.def("swiglu_bwd", &swiglu_bwd);
    m.def("gelu", &gelu);
    m.def("gelu_bwd", &gelu_bwd);
    m.def("gelu_bwd_slabs", &gelu_bwd_slabs);
    m.def("rmsnorm", &rmsnorm);
    m.def("rmsnorm_bwd", &rmsnorm_bwd);
    m.def("layernorm", &layernorm);
    m.def("layernorm_bwd", &layernorm_bwd);
    m.def("quantize_rowcol", &quantize_rowcol);
    m.def("gemm_nt", &gemm_nt);
    m.def("group_in_one_launch", &group_in_one_launch);
    m.def("gemm_nt_group", &gemm_nt_group);
    m.def("chain_in_one_launch", &chain_in_one_launch);
    m.def("gemm_nt_chain", &gemm_nt_chain);
    m.def("gemm_layouts", &gemm_layouts);
    m.def("mx_cast", &mx_cast);
    m.def("block_cast", &block_cast);
    m.def("mx_gemm_nt", &mx_gemm_nt);
    m.def("residual_norm", &residual_norm);
    m.def("residual_norm_bwd", &residual_norm_bwd);
    m.def("token_logprobs", &token_logprobs);
    m.def("token_logprobs_bwd", &token_logprobs_bwd);
    m.def("fp4_linear", &fp4_linear);
    m.def("residual_norm_node", &residual_norm_node);
    m.def("token_logprobs_node", &token_logprobs_node);
}
