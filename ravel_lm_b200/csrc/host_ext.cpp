// Python binding of the host calls that run once per decode step or per lookup.
//
// A decode step (RavelLayerCache.step) launches one short kernel; through
// ctypes its Python side -- fourteen argument conversions, the dtype / device /
// layout checks and two output allocations -- took longer than the kernel.
// Here the checks, the allocations (the caching allocator through ATen) and the
// C-ABI call run in C++: the Python caller makes one call.  The lookup entry
// points (tape build, latest-k and segmented-sum forward and backward) get the
// same treatment.
//
// Every function here does exactly what the ctypes path in ravel_memory.py does
// with the same arguments: same entry point of libravel_b200.so, same sizes,
// same stream (the current stream of the tensors' device).  Failure statuses are
// returned to the caller, which raises the library's own errors.  The cache step
// returns None when its arguments are not the common case (the caller then
// takes the fully checked Python path, with its error messages).
//
// The dense operators (fused_linear, layer_norm, distill_topk_loss), the vocabulary's (token_embedding,
// linear_cross_entropy) and the optimizer step (adamw_step) live here whole: argument checks, outputs and
// workspaces, and the autograd node, so that a decoded token's call or a small
// training step is not bound by Python.  Workspaces come from the caching
// allocator on the current stream of the tensors' device.

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/ravel_b200.h"

namespace py = pybind11;

namespace {

int payload_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return RAVEL_F32;
        case at::kBFloat16: return RAVEL_BF16;
        case at::kHalf: return RAVEL_F16;
        case at::kDouble: return RAVEL_F64;
        default: return -1;
    }
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

const void* ptr_or_null(const std::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }

at::Tensor bytes(size_t n, const at::Tensor& like) {
    return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

// RavelLayerCache.step for contiguous CUDA tensors on one device, addresses
// int64 or int32 of one type, payloads in the cache dtype, out None or a
// matching (values, mask) pair.  Returns (values, mask), an int status on a
// library failure, or None for any other argument combination.
py::object cache_step(const at::Tensor& values, const at::Tensor& filled, const at::Tensor& ra, const at::Tensor& wa,
                      const at::Tensor& payloads, const py::object& out) {
    if (!values.is_cuda() || values.dim() != 4 || filled.dim() != 3 || ra.dim() != 2 || wa.dim() != 2 ||
        payloads.dim() != 3)
        return py::none();
    const auto dev = values.device();
    if (filled.device() != dev || ra.device() != dev || wa.device() != dev || payloads.device() != dev)
        return py::none();
    const auto adt = ra.scalar_type();
    if ((adt != at::kLong && adt != at::kInt) || wa.scalar_type() != adt) return py::none();
    const int code = payload_code(values.scalar_type());
    if (code < 0 || payloads.scalar_type() != values.scalar_type() || filled.scalar_type() != at::kBool)
        return py::none();
    if (!values.is_contiguous() || !filled.is_contiguous() || !ra.is_contiguous() || !wa.is_contiguous() ||
        !payloads.is_contiguous())
        return py::none();
    const int64_t B = ra.size(0), C = ra.size(1), A = values.size(2), D = values.size(3);
    if (wa.size(0) != B || wa.size(1) != C || values.size(0) != B || values.size(1) != C || payloads.size(0) != B ||
        payloads.size(1) != C || payloads.size(2) != D || filled.size(0) != B || filled.size(1) != C ||
        filled.size(2) != A)
        return py::none();
    at::Tensor vals, mask;
    if (out.is_none()) {
        vals = at::empty({B, C, D}, values.options());
        mask = at::empty({B, C}, filled.options());
    } else {
        if (!py::isinstance<py::tuple>(out) && !py::isinstance<py::list>(out)) return py::none();
        const py::sequence seq = out.cast<py::sequence>();
        if (seq.size() != 2 || !THPVariable_Check(seq[0].ptr()) || !THPVariable_Check(seq[1].ptr()))
            return py::none();
        vals = THPVariable_Unpack(seq[0].ptr());
        mask = THPVariable_Unpack(seq[1].ptr());
        if (vals.dim() != 3 || vals.size(0) != B || vals.size(1) != C || vals.size(2) != D ||
            vals.scalar_type() != values.scalar_type() || vals.device() != dev || !vals.is_contiguous() ||
            mask.dim() != 2 || mask.size(0) != B || mask.size(1) != C || mask.scalar_type() != at::kBool ||
            mask.device() != dev || !mask.is_contiguous())
            return py::none();
    }
    const int rc = ravel_cache_step(values.data_ptr(), static_cast<uint8_t*>(filled.data_ptr()), ra.data_ptr(),
                                    wa.data_ptr(), adt == at::kLong ? RAVEL_I64 : RAVEL_I32, payloads.data_ptr(),
                                    code, B, C, A, D, vals.data_ptr(), static_cast<uint8_t*>(mask.data_ptr()),
                                    stream_of(values));
    if (rc != RAVEL_OK) return py::int_(rc);
    return py::make_tuple(vals, mask);
}

// ravel_tape_build into a new tape and a scratch buffer sized for a lookup of
// payload width D, dtype code dcode and k.  Returns (status, tape, scratch).
std::tuple<int, at::Tensor, at::Tensor> tape_build(const at::Tensor& w, const std::optional<at::Tensor>& r, int code,
                                                   const std::optional<at::Tensor>& mask, int64_t A, int flags,
                                                   int64_t D, int64_t k, int dcode) {
    const int64_t B = w.size(0), T = w.size(1), C = w.size(2);
    const size_t tb = ravel_tape_bytes(B, T, C, A, flags), sb = ravel_scratch_bytes(B, T, C, D, A, k, dcode, flags);
    at::Tensor tape = bytes(tb, w), scratch = bytes(sb, w);
    const int rc = ravel_tape_build(w.data_ptr(), ptr_or_null(r), code,
                                    static_cast<const uint8_t*>(ptr_or_null(mask)), B, T, C, A, flags,
                                    tape.data_ptr(), tb, scratch.data_ptr(), sb, stream_of(w));
    return {rc, tape, scratch};
}

// ravel_latestk_fwd_tape into new [B,T,C,k,D] values and [B,T,C,k] mask.
std::tuple<int, at::Tensor, at::Tensor> latestk_fwd(const at::Tensor& tape, int flags,
                                                    const std::optional<at::Tensor>& r, int code,
                                                    const at::Tensor& p, int64_t B, int64_t T, int64_t C, int64_t A,
                                                    int64_t k) {
    const int64_t D = p.size(-1);
    at::Tensor vals = at::empty({B, T, C, k, D}, p.options());
    at::Tensor mask = at::empty({B, T, C, k}, p.options().dtype(at::kBool));
    const int rc = ravel_latestk_fwd_tape(tape.data_ptr(), flags, ptr_or_null(r), code, p.data_ptr(),
                                          payload_code(p.scalar_type()), B, T, C, D, A, k, vals.data_ptr(),
                                          static_cast<uint8_t*>(mask.data_ptr()), stream_of(p));
    return {rc, vals, mask};
}

// ravel_segsum_fwd_tape into new [B,T,C,D] sums and [B,T,C] mask.
std::tuple<int, at::Tensor, at::Tensor> segsum_fwd(const at::Tensor& tape, int flags,
                                                   const std::optional<at::Tensor>& r, int code, const at::Tensor& p,
                                                   const at::Tensor& scratch, int64_t B, int64_t T, int64_t C,
                                                   int64_t A) {
    const int64_t D = p.size(-1);
    at::Tensor sums = at::empty({B, T, C, D}, p.options());
    at::Tensor mask = at::empty({B, T, C}, p.options().dtype(at::kBool));
    const int rc = ravel_segsum_fwd_tape(tape.data_ptr(), flags, ptr_or_null(r), code, p.data_ptr(),
                                         payload_code(p.scalar_type()), B, T, C, D, A, sums.data_ptr(),
                                         static_cast<uint8_t*>(mask.data_ptr()), scratch.data_ptr(),
                                         static_cast<size_t>(scratch.numel()), stream_of(p));
    return {rc, sums, mask};
}

// ravel_segsum_bwd into a new [B,T,C,D] payload gradient.
std::tuple<int, at::Tensor> segsum_bwd(const at::Tensor& tape, int flags, const std::optional<at::Tensor>& r,
                                       int code, const at::Tensor& g, int64_t B, int64_t T, int64_t C, int64_t A) {
    const int64_t D = g.size(-1);
    const int dcode = payload_code(g.scalar_type());
    const size_t sb = ravel_scratch_bytes(B, T, C, D, A, 1, dcode, flags);
    at::Tensor grad = at::empty({B, T, C, D}, g.options());
    at::Tensor scratch = bytes(sb, g);
    const int rc = ravel_segsum_bwd(tape.data_ptr(), flags, ptr_or_null(r), code, g.data_ptr(), dcode, B, T, C, D, A,
                                    grad.data_ptr(), scratch.data_ptr(), sb, stream_of(g));
    return {rc, grad};
}

// ravel_latestk_bwd into a new payload gradient, or ravel_latestk_bwd_accumulate
// into acc (checked by the caller: contiguous [B,T,C,D] of the gradient dtype).
std::tuple<int, at::Tensor> latestk_bwd(const at::Tensor& tape, int flags, const std::optional<at::Tensor>& r,
                                        int code, const at::Tensor& g, int64_t B, int64_t T, int64_t C, int64_t A,
                                        int64_t k, const std::optional<at::Tensor>& acc) {
    const int64_t D = g.size(-1);
    const int dcode = payload_code(g.scalar_type());
    const size_t sb = ravel_scratch_bytes(B, T, C, D, A, k, dcode, flags);
    at::Tensor grad = acc ? *acc : at::empty({B, T, C, D}, g.options());
    at::Tensor scratch = bytes(sb, g);
    const int rc = (acc ? ravel_latestk_bwd_accumulate : ravel_latestk_bwd)(
        tape.data_ptr(), flags, ptr_or_null(r), code, g.data_ptr(), dcode, B, T, C, D, A, k, grad.data_ptr(),
        scratch.data_ptr(), sb, stream_of(g));
    return {rc, grad};
}

// ------------------------------------------------------------------ dense operators
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

// A failed library call as the Python error _lib.check raises for its status.
void check_status(const char* entry, int rc) {
    if (rc == RAVEL_OK) return;
    const std::string msg =
        std::string(entry) + " failed: " + ravel_status_string(rc) + " (status " + std::to_string(rc) + ")";
    if (rc == RAVEL_ERR_INVALID_ARG || rc == RAVEL_ERR_UNSUPPORTED) throw py::value_error(msg);
    throw std::runtime_error(msg);
}

void require_cuda(const at::Tensor& first, std::initializer_list<const OptTensor*> others) {
    auto cuda = [](const at::Tensor& t) {
        if (!t.is_cuda())
            throw std::runtime_error("ravel_lm_b200 runs on CUDA tensors only (got a " + t.device().str() +
                                     " tensor); there is no CPU fallback");
    };
    cuda(first);
    for (const OptTensor* t : others) {
        if (!t->has_value()) continue;
        cuda(**t);
        if ((*t)->device() != first.device())
            throw std::runtime_error("tensors are on different devices: " + first.device().str() + " and " +
                                     (*t)->device().str());
    }
}

// The backward kernels have no derivative of their own: refuse create_graph rather than return gradients that
// silently lack one.
void once_differentiable(const char* op) {
    if (at::GradMode::is_enabled())
        throw std::runtime_error(std::string(op) + ": the backward pass is not differentiable (create_graph=True)");
}

// Nor is there a forward-mode derivative: refuse a tangent rather than drop it.
void no_tangents(const char* op, std::initializer_list<const OptTensor*> tensors) {
    for (const OptTensor* t : tensors)
        if (t->has_value() && (*t)->_fw_grad(/*level=*/0).defined())
            throw std::runtime_error(std::string(op) + " has no forward-mode derivative");
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// A row-major matrix as the kernels take it: elements of a row adjacent, rows `ld` apart.
struct Rows {
    at::Tensor t;  // holds the memory
    int64_t ld = 0;
};

int64_t leading(const at::Tensor& t) {
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
    return n;
}

// [..., n] as [leading, n] with adjacent elements (a view where the strides allow one).
Rows rows_of(const at::Tensor& x) {
    const int64_t n = x.size(-1), m = leading(x);
    at::Tensor t = x.dim() == 2 ? x : x.reshape({m, n});
    if ((n > 1 && t.stride(1) != 1) || (m > 1 && t.stride(0) < n)) t = t.contiguous();
    return {t, m > 1 ? t.stride(0) : up8(n)};
}

// The same for an operand that TMA reads: 16-byte aligned rows, copied to such a pitch (of a multiple of
// `multiple` elements) when the tensor has none.
Rows tma_rows(const at::Tensor& x, int64_t multiple = 8) {
    Rows r = rows_of(x);
    const int64_t m = r.t.size(0), n = r.t.size(1);
    if (m == 0 || n == 0) return r;
    if (r.ld % 8 == 0 && reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16 == 0) return r;
    const int64_t pitch = (n + multiple - 1) / multiple * multiple;
    Rows p{at::empty({m, pitch}, r.t.options()), pitch};
    check_status("ravel_pad_rows", ravel_pad_rows(r.t.data_ptr(), r.ld, m, n, p.t.data_ptr(), p.ld,
                                                  payload_code(r.t.scalar_type()), stream_of(r.t)));
    return p;
}

// y = residual + act(x W^T + bias); x2 and w2 from tma_rows.  z (when wanted): the sum before
// the activation, rows up8(N) apart.
at::Tensor linear_forward(const Rows& x2, const Rows& w2, int64_t M, int64_t K, int64_t N, const OptTensor& bias,
                          const OptTensor& residual, int act, at::IntArrayRef out_shape, at::Tensor* z) {
    at::Tensor y = at::empty(out_shape, x2.t.options());
    OptTensor b = bias ? OptTensor(bias->contiguous()) : std::nullopt;
    Rows res;
    if (residual) res = rows_of(*residual);
    if (z != nullptr) *z = at::empty({M, up8(N)}, x2.t.options());
    check_status("ravel_matmul",
                 ravel_matmul(x2.t.data_ptr(), x2.ld, 0, w2.t.data_ptr(), w2.ld, 0, M, N, K, ptr_or_null(b),
                              residual ? res.t.data_ptr() : nullptr, res.ld, act, y.data_ptr(), N,
                              z != nullptr ? z->data_ptr() : nullptr, up8(N), payload_code(y.scalar_type()),
                              stream_of(y)));
    return y;
}

struct FusedLinear : public torch::autograd::Function<FusedLinear> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                              const OptTensor& bias, const OptTensor& residual, int64_t act) {
        const int64_t K = x.size(-1), M = leading(x), N = weight.size(0);
        const Rows x2 = tma_rows(x), w2 = tma_rows(weight);
        std::vector<int64_t> shape = x.sizes().vec();
        shape.back() = N;
        // without an activation d z is the output's gradient, and z is not needed
        const bool keep_z = act != RAVEL_ACT_NONE && (x.requires_grad() || weight.requires_grad() ||
                                                      (bias && bias->requires_grad()));
        at::Tensor z;
        at::Tensor y = linear_forward(x2, w2, M, K, N, bias, residual, static_cast<int>(act), shape,
                                      keep_z ? &z : nullptr);
        // the backward of relu settles the signs of sums near zero, bias included
        const bool keep_b = act == RAVEL_ACT_RELU && bias.has_value();
        ctx->save_for_backward({x2.t, w2.t, z, keep_b ? bias->contiguous() : at::Tensor()});
        ctx->saved_data["x_ld"] = x2.ld;
        ctx->saved_data["w_ld"] = w2.ld;
        ctx->saved_data["x_shape"] = x.sizes().vec();
        ctx->saved_data["N"] = N;
        ctx->saved_data["act"] = act;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x2 = saved[0], &w2 = saved[1], &z = saved[2], &bias = saved[3];
        const std::vector<int64_t> x_shape = ctx->saved_data["x_shape"].toIntVector();
        const int64_t x_ld = ctx->saved_data["x_ld"].toInt(), w_ld = ctx->saved_data["w_ld"].toInt();
        const int64_t N = ctx->saved_data["N"].toInt(), K = x_shape.back();
        const int act = static_cast<int>(ctx->saved_data["act"].toInt());
        // the gradients this pass asks for; edges are counted over the tensors that were given
        const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool need_b = has_b && ctx->needs_input_grad(2);
        const bool need_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
        int64_t M = 1;
        for (size_t d = 0; d + 1 < x_shape.size(); ++d) M *= x_shape[d];
        variable_list out(5);
        if (!grads[0].defined()) return out;
        once_differentiable("fused_linear");
        const c10::cuda::CUDAGuard guard(x2.device());
        if (need_r) out[3] = grads[0];
        if (!need_x && !need_w && !need_b) return out;
        const Rows gy = rows_of(grads[0]);
        void* const st = stream_of(gy.t);
        const int dt = payload_code(gy.t.scalar_type());
        const bool products = need_x || need_w;
        // the operand of the products: dy itself, or dz (16 bits, TMA-readable rows)
        Rows dz = gy;
        const bool own_dz = products && (act != RAVEL_ACT_NONE || gy.ld % 8 != 0 ||
                                         reinterpret_cast<uintptr_t>(gy.t.data_ptr()) % 16 != 0);
        if (own_dz) dz = Rows{at::empty({M, up8(N)}, gy.t.options()), up8(N)};
        if (own_dz || need_b) {
            at::Tensor scratch;
            size_t sb = 0;
            if (need_b) {
                out[2] = at::empty({N}, gy.t.options());
                sb = ravel_linear_dz_scratch_bytes(M, N);
                scratch = bytes(sb, gy.t);
            }
            check_status("ravel_linear_dz",
                         ravel_linear_dz(gy.t.data_ptr(), gy.ld, z.defined() ? z.data_ptr() : nullptr, up8(N), act,
                                         own_dz ? dz.t.data_ptr() : nullptr, dz.ld,
                                         need_b ? out[2].data_ptr() : nullptr, M, N, x2.data_ptr(), x_ld,
                                         w2.data_ptr(), w_ld, bias.defined() ? bias.data_ptr() : nullptr, K, dt,
                                         need_b ? scratch.data_ptr() : nullptr, sb, st));
        }
        if (need_x) {
            at::Tensor dx = at::empty(x_shape, gy.t.options());
            check_status("ravel_matmul", ravel_matmul(dz.t.data_ptr(), dz.ld, 0, w2.data_ptr(), w_ld, 1, M, K, N,
                                                      nullptr, nullptr, 0, RAVEL_ACT_NONE, dx.data_ptr(), K, nullptr,
                                                      0, dt, st));
            out[0] = dx;
        }
        if (need_w) {
            at::Tensor dw = at::empty({N, K}, gy.t.options());
            check_status("ravel_matmul", ravel_matmul(dz.t.data_ptr(), dz.ld, 1, x2.data_ptr(), x_ld, 1, N, K, M,
                                                      nullptr, nullptr, 0, RAVEL_ACT_NONE, dw.data_ptr(), K, nullptr,
                                                      0, dt, st));
            out[1] = dw;
        }
        return out;
    }
};

at::Tensor fused_linear(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                        const OptTensor& residual, int64_t act) {
    if (x.dim() < 1 || weight.dim() != 2 || weight.size(1) != x.size(-1))
        throw py::value_error("fused_linear expects x [..., K] and a weight [N, K]");
    const auto dt = x.scalar_type();
    if (dt != at::kBFloat16 && dt != at::kHalf)
        throw py::type_error(std::string("fused_linear takes bfloat16 or float16 tensors, got ") + toString(dt));
    if (weight.scalar_type() != dt || (bias && bias->scalar_type() != dt) || (residual && residual->scalar_type() != dt))
        throw py::type_error("fused_linear expects x, weight, bias and residual of one dtype");
    const int64_t N = weight.size(0);
    if (bias && (bias->dim() != 1 || bias->size(0) != N)) throw py::value_error("bias must have shape [N]");
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = N;
    if (residual && residual->sizes() != at::IntArrayRef(shape))
        throw py::value_error("residual must have the output's shape [..., N]");
    const OptTensor in(x), w(weight);
    no_tangents("fused_linear", {&in, &w, &bias, &residual});
    require_cuda(x, {&w, &bias, &residual});
    const c10::cuda::CUDAGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled() &&
                      (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()) ||
                       (residual && residual->requires_grad()));
    if (grad) return FusedLinear::apply(x, weight, bias, residual, act);
    return linear_forward(tma_rows(x), tma_rows(weight), leading(x), x.size(-1), N, bias, residual,
                          static_cast<int>(act), shape, nullptr);
}

// The element types of LayerNorm and of logits.
int float_code(const at::Tensor& t, const char* what) {
    const int c = payload_code(t.scalar_type());
    if (c != RAVEL_F32 && c != RAVEL_BF16 && c != RAVEL_F16)
        throw py::type_error(std::string(what) + " takes float32, bfloat16 or float16 tensors, got " +
                             toString(t.scalar_type()));
    return c;
}

at::Tensor norm_forward(const Rows& x2, at::IntArrayRef shape, const OptTensor& weight, const OptTensor& bias,
                        double eps, at::Tensor* mean, at::Tensor* rstd) {
    const int64_t M = x2.t.size(0), K = x2.t.size(1);
    at::Tensor y = at::empty(shape, x2.t.options());
    if (mean != nullptr) {
        *mean = at::empty({M}, x2.t.options().dtype(at::kFloat));
        *rstd = at::empty({M}, x2.t.options().dtype(at::kFloat));
    }
    check_status("ravel_layer_norm_fwd",
                 ravel_layer_norm_fwd(x2.t.data_ptr(), x2.ld, ptr_or_null(weight), ptr_or_null(bias),
                                      static_cast<float>(eps), y.data_ptr(),
                                      mean != nullptr ? mean->data_ptr<float>() : nullptr,
                                      rstd != nullptr ? rstd->data_ptr<float>() : nullptr, M, K,
                                      payload_code(y.scalar_type()), stream_of(y)));
    return y;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& weight, const OptTensor& bias,
                              double eps) {
        const Rows x2 = rows_of(x);
        const OptTensor w = weight ? OptTensor(weight->contiguous()) : std::nullopt;
        const OptTensor b = bias ? OptTensor(bias->contiguous()) : std::nullopt;
        at::Tensor mean, rstd;
        at::Tensor y = norm_forward(x2, x.sizes(), w, b, eps, &mean, &rstd);
        ctx->save_for_backward({x2.t, w ? *w : at::Tensor(), mean, rstd});
        ctx->saved_data["ld"] = x2.ld;
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["weight"] = weight.has_value();
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x2 = saved[0], &w = saved[1], &mean = saved[2], &rstd = saved[3];
        const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1);
        const bool need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
        variable_list out(4);
        once_differentiable("layer_norm");
        if (!grads[0].defined() || !(need_x || need_w || need_b)) return out;
        const c10::cuda::CUDAGuard guard(x2.device());
        const int64_t M = x2.size(0), K = x2.size(1);
        const Rows gy = rows_of(grads[0]);
        at::Tensor scratch, dw, db;
        size_t sb = 0;
        if (need_x) out[0] = at::empty(ctx->saved_data["shape"].toIntVector(), x2.options());
        if (need_w || need_b) {  // one pass makes both
            dw = at::empty({K}, x2.options());
            db = at::empty({K}, x2.options());
            sb = ravel_layer_norm_scratch_bytes(M, K);
            scratch = bytes(sb, x2);
        }
        check_status("ravel_layer_norm_bwd",
                     ravel_layer_norm_bwd(x2.data_ptr(), ctx->saved_data["ld"].toInt(),
                                          w.defined() ? w.data_ptr() : nullptr, gy.t.data_ptr(), gy.ld,
                                          mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                          need_x ? out[0].data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
                                          db.defined() ? db.data_ptr() : nullptr, M, K,
                                          payload_code(x2.scalar_type()), sb ? scratch.data_ptr() : nullptr, sb,
                                          stream_of(x2)));
        if (need_w) out[1] = dw;
        if (need_b) out[2] = db;
        return out;
    }
};

at::Tensor layer_norm(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error("layer_norm expects x [..., K] with K >= 1");
    const int64_t K = x.size(-1);
    for (const OptTensor* t : {&weight, &bias})
        if (t->has_value() && ((*t)->dim() != 1 || (*t)->size(0) != K))
            throw py::value_error("layer_norm expects weight and bias of shape [x.shape[-1]]");
    float_code(x, "layer_norm");
    for (const OptTensor* t : {&weight, &bias})
        if (t->has_value() && (*t)->scalar_type() != x.scalar_type())
            throw py::type_error("layer_norm expects x, weight and bias of one dtype");
    const OptTensor in(x);
    no_tangents("layer_norm", {&in, &weight, &bias});
    require_cuda(x, {&weight, &bias});
    const c10::cuda::CUDAGuard guard(x.device());
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
        return LayerNorm::apply(x, weight, bias, eps);
    return norm_forward(rows_of(x), x.sizes(), weight ? OptTensor(weight->contiguous()) : std::nullopt,
                        bias ? OptTensor(bias->contiguous()) : std::nullopt, eps, nullptr, nullptr);
}

// The tensors of a distillation call, and its launch.
struct DistillCall {
    Rows s;
    at::Tensor ids, teacher, losses, stat, scratch, out;
    int64_t R, V, k;
    float tau, weight;
    int reduction, dtype;

    DistillCall(const at::Tensor& logits, const at::Tensor& ids_, const at::Tensor& teacher_, double tau_,
                double weight_, int64_t reduction_)
        : s(rows_of(logits)), ids(ids_.contiguous()), teacher(teacher_.contiguous()), R(s.t.size(0)), V(s.t.size(1)),
          k(ids_.size(-1)), tau(static_cast<float>(tau_)), weight(static_cast<float>(weight_)),
          reduction(static_cast<int>(reduction_)), dtype(payload_code(logits.scalar_type())) {}

    int ids_code() const { return ids.scalar_type() == at::kLong ? RAVEL_I64 : RAVEL_I32; }

    // losses (and their reduction); stat is kept and grad written where wanted.
    at::Tensor forward(at::IntArrayRef rows_shape, bool keep, const at::Tensor& grad) {
        const auto f32 = s.t.options().dtype(at::kFloat);
        losses = at::empty(rows_shape, f32);
        if (keep) stat = at::empty({R, 2}, f32);
        const size_t sb = reduction == RAVEL_REDUCE_MEAN ? ravel_distill_topk_scratch_bytes(R) : 0;
        if (sb) scratch = bytes(sb, s.t);
        if (reduction != RAVEL_REDUCE_NONE) out = at::empty({}, f32);
        check_status("ravel_distill_topk_fwd",
                     ravel_distill_topk_fwd(s.t.data_ptr(), s.ld, ids.data_ptr(), ids_code(), teacher.data_ptr(),
                                            payload_code(teacher.scalar_type()), R, V, k, tau, weight, reduction,
                                            losses.data_ptr<float>(), keep ? stat.data_ptr<float>() : nullptr,
                                            out.defined() ? out.data_ptr<float>() : nullptr,
                                            grad.defined() ? grad.data_ptr() : nullptr, dtype,
                                            sb ? scratch.data_ptr() : nullptr, sb, stream_of(s.t)));
        return reduction == RAVEL_REDUCE_NONE ? losses : out;
    }
};

struct DistillTopk : public torch::autograd::Function<DistillTopk> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids,
                              const at::Tensor& teacher, double tau, double weight, int64_t reduction) {
        DistillCall c(logits, ids, teacher, tau, weight, reduction);
        // The gradient for an upstream gradient of 1 while the rows are in cache: a training step
        // then reads the logits from memory once.  Not for float16, where it may underflow before
        // the loss scaling of the upstream gradient reaches it, nor for single rows' losses, whose
        // upstream gradients are rarely 1.
        at::Tensor unit;
        if (reduction != RAVEL_REDUCE_NONE && c.dtype != RAVEL_F16) unit = at::empty(logits.sizes(), c.s.t.options());
        const auto sizes = logits.sizes();
        at::Tensor loss = c.forward(sizes.slice(0, sizes.size() - 1), true, unit);
        ctx->save_for_backward({c.s.t, c.ids, c.teacher, c.stat, c.scratch});
        if (unit.defined()) ctx->saved_data["unit"] = unit;
        ctx->saved_data["ld"] = c.s.ld;
        ctx->saved_data["shape"] = sizes.vec();
        ctx->saved_data["tau"] = tau;
        ctx->saved_data["weight"] = weight;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &s = saved[0], &ids = saved[1], &teacher = saved[2], &stat = saved[3], &scratch = saved[4];
        variable_list out(6);
        if (!grads[0].defined()) return out;
        once_differentiable("distill_topk_loss");
        const c10::cuda::CUDAGuard guard(s.device());
        // The forward's gradient is given away once; a second backward pass writes a new one.
        at::Tensor grad;
        const auto it = ctx->saved_data.find("unit");
        const bool unit = it != ctx->saved_data.end();
        if (unit) {
            grad = it->second.toTensor();
            ctx->saved_data.erase(it);
        } else {
            grad = at::empty(ctx->saved_data["shape"].toIntVector(), s.options());
        }
        const at::Tensor up = grads[0].contiguous();
        check_status(
            "ravel_distill_topk_bwd",
            ravel_distill_topk_bwd(s.data_ptr(), ctx->saved_data["ld"].toInt(), ids.data_ptr(),
                                   ids.scalar_type() == at::kLong ? RAVEL_I64 : RAVEL_I32, teacher.data_ptr(),
                                   payload_code(teacher.scalar_type()), s.size(0), s.size(1), ids.size(-1),
                                   static_cast<float>(ctx->saved_data["tau"].toDouble()),
                                   static_cast<float>(ctx->saved_data["weight"].toDouble()),
                                   static_cast<int>(ctx->saved_data["reduction"].toInt()), stat.data_ptr<float>(),
                                   scratch.defined() ? scratch.data_ptr() : nullptr,
                                   up.data_ptr<float>(), unit ? 1 : 0, grad.data_ptr(),
                                   payload_code(s.scalar_type()), stream_of(s)));
        out[0] = grad;
        return out;
    }
};

at::Tensor distill_topk_loss(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher, double tau,
                             double weight, int64_t reduction) {
    if (logits.dim() < 1 || logits.size(-1) < 1)
        throw py::value_error("distill_topk_loss expects logits [..., V] with V >= 1");
    if (ids.dim() != logits.dim() || ids.sizes() != teacher.sizes() ||
        ids.sizes().slice(0, ids.dim() - 1) != logits.sizes().slice(0, logits.dim() - 1))
        throw py::value_error("teacher_ids and teacher_logits must both be [..., k] with the logits' leading dimensions");
    if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong)
        throw py::type_error("teacher_ids must be int32 or int64");
    float_code(logits, "distill_topk_loss");
    float_code(teacher, "distill_topk_loss");
    if (!(tau > 0.0) || !std::isfinite(tau)) throw py::value_error("temperature must be positive and finite");
    if (teacher.requires_grad() && at::GradMode::is_enabled())
        throw py::value_error("teacher_logits must not require a gradient (detach them)");
    const OptTensor s(logits), i(ids), t(teacher);
    no_tangents("distill_topk_loss", {&s, &t});
    require_cuda(logits, {&i, &t});
    const c10::cuda::CUDAGuard guard(logits.device());
    if (at::GradMode::is_enabled() && logits.requires_grad())
        return DistillTopk::apply(logits, ids, teacher, tau, weight, reduction);
    DistillCall c(logits, ids, teacher, tau, weight, reduction);
    return c.forward(logits.sizes().slice(0, logits.dim() - 1), false, at::Tensor());
}

// ------------------------------------------------------------------ the vocabulary's two ends
int index_code(const at::Tensor& t, const char* what) {
    if (t.scalar_type() == at::kLong) return RAVEL_I64;
    if (t.scalar_type() == at::kInt) return RAVEL_I32;
    throw py::type_error(std::string(what) + " must be int32 or int64");
}

at::Tensor embedding_forward(const at::Tensor& ids, const Rows& w, double scale) {
    std::vector<int64_t> shape = ids.sizes().vec();
    const int64_t V = w.t.size(0), K = w.t.size(1);
    shape.push_back(K);
    at::Tensor y = at::empty(shape, w.t.options());
    check_status("ravel_embedding_fwd",
                 ravel_embedding_fwd(ids.data_ptr(), index_code(ids, "ids"), w.t.data_ptr(), w.ld, ids.numel(), V, K,
                                     static_cast<float>(scale), y.data_ptr(), payload_code(y.scalar_type()),
                                     stream_of(y)));
    return y;
}

struct TokenEmbedding : public torch::autograd::Function<TokenEmbedding> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& weight, double scale,
                              int64_t padding) {
        at::Tensor y = embedding_forward(ids, rows_of(weight), scale);
        ctx->save_for_backward({ids});
        ctx->saved_data["V"] = weight.size(0);
        ctx->saved_data["K"] = weight.size(1);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const at::Tensor& ids = saved[0];
        variable_list out(4);
        if (!grads[0].defined()) return out;
        once_differentiable("token_embedding");
        const c10::cuda::CUDAGuard guard(ids.device());
        const int64_t V = ctx->saved_data["V"].toInt(), K = ctx->saved_data["K"].toInt(), N = ids.numel();
        const Rows gy = rows_of(grads[0]);
        at::Tensor dw = at::empty({V, K}, gy.t.options());
        const size_t sb = ravel_embedding_scratch_bytes(N, V, K);
        at::Tensor scratch;
        if (sb > 0) scratch = bytes(sb, gy.t);
        check_status("ravel_embedding_bwd",
                     ravel_embedding_bwd(ids.data_ptr(), index_code(ids, "ids"), gy.t.data_ptr(), gy.ld, N, V, K,
                                         static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                         ctx->saved_data["padding"].toInt(), dw.data_ptr(),
                                         payload_code(dw.scalar_type()), sb > 0 ? scratch.data_ptr() : nullptr, sb,
                                         stream_of(gy.t)));
        out[1] = dw;
        return out;
    }
};

at::Tensor token_embedding(const at::Tensor& ids, const at::Tensor& weight, double scale,
                           std::optional<int64_t> padding_idx) {
    if (weight.dim() != 2 || weight.size(0) < 1)
        throw py::value_error("token_embedding expects a weight [V, K] with V >= 1");
    index_code(ids, "ids");
    float_code(weight, "token_embedding");
    if (!std::isfinite(static_cast<float>(scale))) throw py::value_error("scale must be finite (in float32)");
    const int64_t V = weight.size(0);
    int64_t padding = -1;
    if (padding_idx) {
        padding = *padding_idx < 0 ? *padding_idx + V : *padding_idx;
        if (padding < 0 || padding >= V) throw py::value_error("padding_idx must lie in the vocabulary");
    }
    const OptTensor i(ids), w(weight);
    no_tangents("token_embedding", {&w});
    require_cuda(ids, {&w});
    const c10::cuda::CUDAGuard guard(weight.device());
    const at::Tensor idc = ids.contiguous();
    if (at::GradMode::is_enabled() && weight.requires_grad())
        return TokenEmbedding::apply(idc, weight, scale, padding);
    return embedding_forward(idc, rows_of(weight), scale);
}

// A cross entropy call's forward, and the gradients' float32 sums: slabs of d x, slabs of d W and their factor in one
// allocation.
struct CrossEntropyCall {
    Rows w;
    int64_t M, K, V;
    int dtype;
    at::Tensor out, scratch, sums;
    int64_t nx = 0;  // floats of d x's slabs
    float *slabs_x = nullptr, *slabs_w = nullptr, *factor = nullptr;

    // w: rows that TMA can read, of K elements and perhaps padding
    CrossEntropyCall(const Rows& w_, int64_t M_, int64_t K_, int64_t V_)
        : w(w_), M(M_), K(K_), V(V_), dtype(payload_code(w_.t.scalar_type())) {}

    void make_sums(bool need_x, bool need_w) {
        int64_t sizes[3];
        check_status("ravel_linear_ce_slabs", ravel_linear_ce_slabs(M, K, V, sizes));
        const int64_t n = need_x ? sizes[0] * M * sizes[2] : 0, nw = need_w ? sizes[1] * V * sizes[2] : 0;
        hold(at::empty({n + nw + 1}, w.t.options().dtype(at::kFloat)), n);
    }
    void hold(const at::Tensor& t, int64_t n) {  // rows of whole 4 floats: every slab is 16-byte aligned
        sums = t;
        nx = n;
        const int64_t all = sums.numel() - 1;
        float* const p = sums.data_ptr<float>();
        slabs_x = nx > 0 ? p : nullptr;
        slabs_w = all > nx ? p + nx : nullptr;
        factor = p + all;
    }

    // keep: what the backward of single rows' losses needs stays in scratch
    at::Tensor forward(const Rows& x, const at::Tensor& targets, int64_t ignore, int reduction, bool need_x, bool need_w,
                       bool keep, at::IntArrayRef rows_shape) {
        const auto f32 = w.t.options().dtype(at::kFloat);
        const bool reduced = reduction != RAVEL_REDUCE_NONE, grads = reduced && (need_x || need_w);
        out = reduced ? at::empty({}, f32) : at::empty(rows_shape, f32);
        if (grads) make_sums(need_x, need_w);
        const size_t sb = ravel_linear_ce_scratch_bytes(M, K, V);
        const size_t wb = ravel_linear_ce_work_bytes(M, K, V, grads, dtype);
        // a reduced loss needs nothing of it later: losses, scratch and work in one
        const size_t lb = reduced ? (static_cast<size_t>(M) * 4 + 255) / 256 * 256 : 0;
        at::Tensor work = bytes(lb + (keep ? 0 : sb) + wb, w.t);
        char* const p = static_cast<char*>(work.data_ptr());
        if (keep) scratch = bytes(sb, w.t);
        check_status("ravel_linear_ce_fwd",
                     ravel_linear_ce_fwd(x.t.data_ptr(), x.ld, w.t.data_ptr(), w.ld, targets.data_ptr(),
                                         index_code(targets, "targets"), M, K, V, ignore, reduction, keep,
                                         reduced ? reinterpret_cast<float*>(p) : out.data_ptr<float>(),
                                         reduced ? out.data_ptr<float>() : nullptr, factor, slabs_x, slabs_w, dtype,
                                         keep ? scratch.data_ptr() : p + lb, sb, p + lb + (keep ? 0 : sb), wb,
                                         stream_of(w.t)));
        return out;
    }
};

struct LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                              const at::Tensor& targets, int64_t ignore, int64_t reduction) {
        // A reduced loss's gradients are made here, a piece of the rows at a time, while their logits exist, up to a
        // factor that the backward applies: float32 sums, so that nothing depends on the size of the upstream gradient.
        CrossEntropyCall c(tma_rows(weight, 64), leading(x), weight.size(1), weight.size(0));
        const bool reduced = reduction != RAVEL_REDUCE_NONE;
        at::Tensor loss = c.forward(rows_of(x), targets, ignore, static_cast<int>(reduction), x.requires_grad(),
                                    weight.requires_grad(), !reduced, targets.sizes());
        ctx->save_for_backward({c.sums, reduced ? at::Tensor() : c.w.t, c.scratch});
        ctx->saved_data["nx"] = c.nx;
        ctx->saved_data["ld"] = c.w.ld;
        ctx->saved_data["M"] = c.M;
        ctx->saved_data["K"] = c.K;
        ctx->saved_data["V"] = c.V;
        ctx->saved_data["dtype"] = static_cast<int64_t>(c.dtype);
        ctx->saved_data["x_shape"] = x.sizes().vec();
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        variable_list out(5);
        if (!grads[0].defined()) return out;
        once_differentiable("linear_cross_entropy");
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        if (!need_x && !need_w) return out;
        const at::Tensor up = grads[0].contiguous();
        const c10::cuda::CUDAGuard guard(up.device());
        const int64_t M = ctx->saved_data["M"].toInt(), K = ctx->saved_data["K"].toInt(), V = ctx->saved_data["V"].toInt();
        const int dtype = static_cast<int>(ctx->saved_data["dtype"].toInt());
        void* const st = stream_of(up);
        const bool reduced = saved[0].defined();
        CrossEntropyCall c(Rows{reduced ? saved[0] : saved[1], ctx->saved_data["ld"].toInt()}, M, K, V);
        if (reduced) {  // which sums there are was settled by the forward
            c.hold(saved[0], ctx->saved_data["nx"].toInt());
        } else {
            c.make_sums(need_x, need_w);
            at::Tensor scratch = saved[2];
            const size_t wb = ravel_linear_ce_work_bytes(M, K, V, 1, dtype);
            at::Tensor work = bytes(wb, up);
            check_status("ravel_linear_ce_grad",
                         ravel_linear_ce_grad(c.w.t.data_ptr(), c.w.ld, up.data_ptr<float>(), M, K, V,
                                              c.factor, c.slabs_x, c.slabs_w, dtype, scratch.data_ptr(),
                                              static_cast<size_t>(scratch.numel()), work.data_ptr(), wb, st));
        }
        const auto like = up.options().dtype(dtype == RAVEL_F16 ? at::kHalf : at::kBFloat16);
        if (need_x) out[0] = at::empty(ctx->saved_data["x_shape"].toIntVector(), like);
        if (need_w) out[1] = at::empty({V, K}, like);
        check_status("ravel_linear_ce_bwd",
                     ravel_linear_ce_bwd(c.slabs_x, c.slabs_w, reduced ? up.data_ptr<float>() : nullptr, c.factor, M, K, V,
                                         need_x ? out[0].data_ptr() : nullptr, need_w ? out[1].data_ptr() : nullptr,
                                         dtype, st));
        return out;
    }
};

at::Tensor linear_cross_entropy(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, int64_t ignore,
                                int64_t reduction) {
    if (x.dim() < 1 || weight.dim() != 2 || weight.size(1) != x.size(-1) || weight.size(0) < 1 || weight.size(1) < 1)
        throw py::value_error("linear_cross_entropy expects x [..., K] and a weight [V, K], V and K at least 1");
    if (targets.sizes() != x.sizes().slice(0, x.dim() - 1))
        throw py::value_error("targets must have x's leading dimensions");
    const auto dt = x.scalar_type();
    if (dt != at::kBFloat16 && dt != at::kHalf)
        throw py::type_error(std::string("linear_cross_entropy takes bfloat16 or float16 tensors, got ") + toString(dt));
    if (weight.scalar_type() != dt) throw py::type_error("linear_cross_entropy expects x and weight of one dtype");
    index_code(targets, "targets");
    const OptTensor in(x), w(weight), t(targets);
    no_tangents("linear_cross_entropy", {&in, &w});
    require_cuda(x, {&w, &t});
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor tc = targets.contiguous();
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad()))
        return LinearCrossEntropy::apply(x, weight, tc, ignore, reduction);
    CrossEntropyCall c(tma_rows(weight, 64), leading(x), weight.size(1), weight.size(0));
    return c.forward(rows_of(x), tc, ignore, static_cast<int>(reduction), false, false, false, tc.sizes());
}

// ------------------------------------------------------------------ the optimizer step
using TensorList = std::vector<at::Tensor>;
using OptTensorList = std::optional<TensorList>;

void written(const at::Tensor& t) {  // autograd counts writes in place
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::string at_place(const char* what, size_t i) { return std::string(what) + "[" + std::to_string(i) + "]"; }

at::Tensor global_norm(const TensorList& tensors) {
    if (tensors.empty()) throw py::value_error("global_norm expects at least one tensor");
    for (const at::Tensor& t : tensors) float_code(t, "global_norm");
    for (const at::Tensor& t : tensors) {
        const OptTensor o(t);
        require_cuda(tensors[0], {&o});
    }
    const c10::cuda::CUDAGuard guard(tensors[0].device());
    std::vector<at::ScalarType> types;
    for (const at::Tensor& t : tensors)
        if (std::find(types.begin(), types.end(), t.scalar_type()) == types.end()) types.push_back(t.scalar_type());
    at::Tensor norms = at::empty({static_cast<int64_t>(types.size())}, tensors[0].options().dtype(at::kDouble));
    TensorList held;
    for (size_t k = 0; k < types.size(); ++k) {
        std::vector<ravel_adamw_tensor> list;
        const at::Tensor* first = nullptr;
        for (const at::Tensor& t : tensors) {
            if (t.scalar_type() != types[k]) continue;
            held.push_back(t.contiguous());
            if (first == nullptr) first = &t;
            list.push_back({nullptr, held.back().data_ptr(), nullptr, nullptr, nullptr, nullptr, nullptr, t.numel()});
        }
        const int64_t count = static_cast<int64_t>(list.size());
        const size_t sb = ravel_grad_norm_scratch_bytes(list.data(), count);
        at::Tensor scratch = bytes(sb, *first);
        check_status("ravel_grad_norm",
                     ravel_grad_norm(list.data(), count, payload_code(types[k]), norms.data_ptr<double>() + k,
                                     scratch.data_ptr(), sb, stream_of(*first)));
    }
    return types.size() == 1 ? norms[0] : at::norm(norms);
}

OptTensor adamw_step(const TensorList& params, const TensorList& grads, const TensorList& avgs, const TensorList& sqs,
                     const at::Tensor& step, const OptTensorList& masters, const OptTensorList& avg_exps,
                     const OptTensorList& sq_exps, double lr, const OptTensor& lr_tensor, double beta1, double beta2,
                     double eps, double weight_decay, std::optional<double> max_norm, const OptTensor& norm,
                     bool positive) {
    const size_t n = params.size();
    if (n == 0) throw py::value_error("adamw_step expects at least one tensor");
    if (grads.size() != n || avgs.size() != n || sqs.size() != n || (masters && masters->size() != n) ||
        (avg_exps && avg_exps->size() != n) || (sq_exps && sq_exps->size() != n))
        throw py::value_error("adamw_step expects lists of one length");
    if (avg_exps.has_value() != sq_exps.has_value())
        throw py::value_error("exp_avg_exponents and exp_avg_sq_exponents come together (8-bit states)");
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
        throw py::value_error("betas must lie in [0, 1)");
    if (!(eps >= 0.0) || !(weight_decay >= 0.0) || (!lr_tensor && !(lr >= 0.0)))
        throw py::value_error("lr, eps and weight_decay must not be negative");
    if (max_norm && !(*max_norm > 0.0)) throw py::value_error("max_norm must be positive");
    if (norm && !max_norm) throw py::value_error("norm is used with max_norm only");
    if (positive && !avg_exps) throw py::value_error("positive_exp_avg_sq is for 8-bit states only");
    const at::Tensor& first = params[0];
    const auto dt = first.scalar_type();
    const bool eight = avg_exps.has_value(), half = dt != at::kFloat;
    float_code(first, "adamw_step");
    if (half != masters.has_value())
        throw py::value_error("16-bit parameters need float32 masters, and float32 parameters take none");
    if (step.scalar_type() != at::kLong || step.numel() != 1) throw py::type_error("step must be one int64");
    if (lr_tensor && (lr_tensor->scalar_type() != at::kFloat || lr_tensor->numel() != 1))
        throw py::type_error("an lr tensor must be one float32");
    if (norm && (norm->scalar_type() != at::kDouble || norm->numel() != 1))
        throw py::type_error("norm must be one float64 (global_norm's)");
    auto check = [&](const char* what, size_t i, const at::Tensor& t, at::ScalarType type, int64_t size) {
        if (t.numel() != size) throw py::value_error(at_place(what, i) + " has the wrong number of elements");
        if (t.scalar_type() != type)
            throw py::type_error(at_place(what, i) + " must be " + toString(type) + ", got " + toString(t.scalar_type()));
        if (!t.is_contiguous()) throw py::value_error(at_place(what, i) + " must be contiguous");
    };
    const auto state = eight ? at::kByte : at::kFloat;
    for (size_t i = 0; i < n; ++i) {
        const int64_t size = params[i].numel();
        check("params", i, params[i], dt, size);
        if (grads[i].sizes() != params[i].sizes()) throw py::value_error(at_place("grads", i) + " must have its parameter's shape");
        if (grads[i].is_sparse()) throw py::value_error(at_place("grads", i) + " must be dense");
        if (grads[i].scalar_type() != dt) throw py::type_error(at_place("grads", i) + " must have its parameter's dtype");
        check("exp_avgs", i, avgs[i], state, size);
        check("exp_avg_sqs", i, sqs[i], state, size);
        if (half) check("masters", i, (*masters)[i], at::kFloat, size);
        if (eight) {
            check("exp_avg_exponents", i, (*avg_exps)[i], at::kChar, (size + 255) / 256);
            check("exp_avg_sq_exponents", i, (*sq_exps)[i], at::kChar, (size + 255) / 256);
        }
    }
    {
        std::vector<const void*> seen;
        for (const at::Tensor& t : params)
            if (t.numel() > 0) seen.push_back(t.data_ptr());
        std::sort(seen.begin(), seen.end());
        if (std::adjacent_find(seen.begin(), seen.end()) != seen.end())
            throw py::value_error("adamw_step: a parameter appears twice");
    }
    const OptTensor st(step);
    require_cuda(first, {&st, &lr_tensor, &norm});
    auto same_device = [&](const TensorList& l) {
        for (const at::Tensor& t : l)
            if (t.device() != first.device()) {
                const OptTensor o(t);
                require_cuda(first, {&o});
            }
    };
    for (const TensorList* l : {&params, &grads, &avgs, &sqs}) same_device(*l);
    for (const OptTensorList* l : {&masters, &avg_exps, &sq_exps})
        if (l->has_value()) same_device(**l);
    const c10::cuda::CUDAGuard guard(first.device());
    TensorList held;  // gradients laid out otherwise
    std::vector<ravel_adamw_tensor> list(n);
    for (size_t i = 0; i < n; ++i) {
        const at::Tensor* g = &grads[i];
        if (!g->is_contiguous()) {
            held.push_back(g->contiguous());
            g = &held.back();
        }
        list[i] = {params[i].data_ptr(), g->data_ptr(), half ? (*masters)[i].data_ptr<float>() : nullptr,
                   avgs[i].data_ptr(), sqs[i].data_ptr(),
                   eight ? static_cast<signed char*>((*avg_exps)[i].data_ptr()) : nullptr,
                   eight ? static_cast<signed char*>((*sq_exps)[i].data_ptr()) : nullptr, params[i].numel()};
    }
    at::Tensor norm32;
    if (max_norm) norm32 = at::empty({}, at::TensorOptions().device(first.device()).dtype(at::kFloat));
    const size_t sb = ravel_adamw_scratch_bytes(list.data(), static_cast<int64_t>(n), max_norm.value_or(0.0));
    at::Tensor scratch = bytes(sb, first);
    check_status("ravel_adamw",
                 ravel_adamw(list.data(), static_cast<int64_t>(n), payload_code(dt),
                             eight ? (positive ? 8 | RAVEL_STATE_POSITIVE : 8) : 32,
                             step.data_ptr<int64_t>(), lr, lr_tensor ? lr_tensor->data_ptr<float>() : nullptr, beta1,
                             beta2, eps, weight_decay, max_norm.value_or(0.0), norm ? norm->data_ptr<double>() : nullptr,
                             max_norm ? norm32.data_ptr<float>() : nullptr, scratch.data_ptr(), sb, stream_of(first)));
    written(step);
    for (size_t i = 0; i < n; ++i) {
        written(params[i]);
        written(avgs[i]);
        written(sqs[i]);
        if (half) written((*masters)[i]);
        if (eight) written((*avg_exps)[i]), written((*sq_exps)[i]);
    }
    return max_norm ? OptTensor(norm32) : std::nullopt;
}

at::Tensor state_values(const at::Tensor& codes, const at::Tensor& exponents, bool is_signed, bool half) {
    if (codes.scalar_type() != at::kByte || exponents.scalar_type() != at::kChar)
        throw py::type_error("state_values expects uint8 codes and int8 exponents");
    if (exponents.numel() != (codes.numel() + 255) / 256)
        throw py::value_error("state_values expects one exponent per block of 256 codes");
    const OptTensor e(exponents);
    require_cuda(codes, {&e});
    const c10::cuda::CUDAGuard guard(codes.device());
    const at::Tensor c = codes.contiguous(), x = exponents.contiguous();
    at::Tensor out = at::empty(codes.sizes(), codes.options().dtype(half ? at::kBFloat16 : at::kFloat));
    check_status("ravel_state_values",
                 ravel_state_values(c.data_ptr(), static_cast<const signed char*>(x.data_ptr()), c.numel(),
                                    is_signed ? 1 : 0, out.data_ptr(), half ? RAVEL_BF16 : RAVEL_F32, stream_of(out)));
    return out;
}

}  // namespace

PYBIND11_MODULE(_ravel_host, m) {
    m.doc() = "C++ host calls of libravel_b200 for the per-step Python paths";
    m.def("cache_step", &cache_step);
    m.def("tape_build", &tape_build);
    m.def("latestk_fwd", &latestk_fwd);
    m.def("segsum_fwd", &segsum_fwd);
    m.def("segsum_bwd", &segsum_bwd);
    m.def("latestk_bwd", &latestk_bwd);
    m.def("fused_linear", &fused_linear);
    m.def("layer_norm", &layer_norm);
    m.def("distill_topk_loss", &distill_topk_loss);
    m.def("token_embedding", &token_embedding);
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("global_norm", &global_norm);
    m.def("adamw_step", &adamw_step);
    m.def("state_values", &state_values);
}
