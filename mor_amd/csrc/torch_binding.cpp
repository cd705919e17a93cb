// C++ registrations of the `mor` operators (the reference's 14, and those on the MX wire format at the end) for the CUDA
// dispatch key (which HIP tensors use under ROCm): the host launchers of the reference (mor/csrc/cuda/fake_quantize.cu,
// "FQ": fake_quantize_cuda :1839-1871, _no_alloc :1876-1907, quant_dequant / e4m3_with_e8_scale :1909-2011, block scaling
// :2013-2230, e8mx :2232-2397, channel scaling :2431-2660, TORCH_LIBRARY_IMPL :2663-2678) rewritten as checks +
// allocations + one call into the C ABI of libmor_hip.so.  The schemas are defined by mor_amd/ops.py; this file only provides faster implementations than
// the Python ones (a few microseconds per call instead of ~14).  It contains no kernels and no arithmetic.
#include <torch/library.h>
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>

#include "../../include/mor_hip.h"

namespace {

// set through mor_torch_set_flags (mor.ops.set_flavour); per host thread, so that a thread that switches the flavour
// for a debugging session does not change the results of the others
thread_local uint32_t g_flags = MOR_FLAG_DEFAULT;

void check(int rc) { TORCH_CHECK(rc == 0, "mor_hip: ", mor_last_error()); }

void check_input(const at::Tensor& t, at::ScalarType dtype, int64_t rows, int64_t cols, const char* what) {
    TORCH_CHECK(t.scalar_type() == dtype, "mor: ", what, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, "mor: ", what, " must have shape (", rows, ", ", cols,
                "), got ", t.sizes());
    TORCH_CHECK(t.is_cuda(), "mor: ", what, " must be a GPU tensor");
}

void check_blocks(int64_t bx, int64_t by) { TORCH_CHECK(bx > 0 && by > 0, "mor: block dims must be positive, got (", bx, ", ", by, ")"); }

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

std::vector<at::Tensor> fake_quantize(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y,
                                      double clamp_threshold, int64_t mode, int64_t sf_type) {
    check_input(input, at::kBFloat16, dim_x, dim_y, "input");
    check_blocks(block_x, block_y);
    const at::Tensor x = input.contiguous();
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor out = at::empty_like(x);
    at::Tensor meta = at::empty({cdiv(dim_x, block_x), cdiv(dim_y, block_y)}, x.options().dtype(at::kInt));
    check(mor_fake_quantize(x.data_ptr(), out.data_ptr(), meta.data_ptr<int32_t>(), dim_x, dim_y, block_x, block_y,
                            clamp_threshold, mode, sf_type, g_flags, stream_of(x)));
    return {out, meta};
}

at::Tensor fake_quantize_no_alloc(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y,
                                  double clamp_threshold, int64_t mode, int64_t sf_type, at::Tensor result) {
    check_input(input, at::kBFloat16, dim_x, dim_y, "input");
    check_input(result, at::kBFloat16, dim_x, dim_y, "result");
    TORCH_CHECK(result.is_contiguous(), "mor: result must be contiguous");
    check_blocks(block_x, block_y);
    const at::Tensor x = input.contiguous();
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor meta = at::empty({cdiv(dim_x, block_x), cdiv(dim_y, block_y)}, x.options().dtype(at::kInt));
    check(mor_fake_quantize(x.data_ptr(), result.data_ptr(), meta.data_ptr<int32_t>(), dim_x, dim_y, block_x, block_y,
                            clamp_threshold, mode, sf_type, g_flags, stream_of(x)));
    return meta;
}

std::vector<at::Tensor> scaling(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y,
                                double e4m3_threshold, int64_t ss_mode, bool channel, bool inplace) {
    check_input(input, at::kBFloat16, dim_x, dim_y, "input");
    check_blocks(block_x, block_y);
    TORCH_CHECK(dim_x % block_x == 0 && dim_y % block_y == 0, "mor: block (", block_x, ", ", block_y,
                ") does not divide the tensor (", dim_x, ", ", dim_y, ")");
    at::Tensor x = input.contiguous();
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor out = inplace ? x : at::empty_like(x);
    const auto i32 = x.options().dtype(at::kInt), f32 = x.options().dtype(at::kFloat);
    at::Tensor meta = at::empty({1}, i32), gamax = at::empty({1}, f32), gnnz = at::empty({1}, i32), gerr = at::empty({1}, f32);
    const size_t nbytes = mor_workspace_bytes(channel ? MOR_OP_CHANNEL_SCALING : MOR_OP_BLOCK_SCALING, dim_x, dim_y, block_x, block_y);
    at::Tensor ws = at::empty({(int64_t)nbytes}, x.options().dtype(at::kByte));
    check(mor_block_scaling(x.data_ptr(), out.data_ptr(), meta.data_ptr<int32_t>(), gamax.data_ptr<float>(), gnnz.data_ptr<int32_t>(),
                            gerr.data_ptr<float>(), dim_x, dim_y, block_x, block_y, e4m3_threshold, ss_mode, channel ? 1 : 0,
                            ws.data_ptr(), nbytes, g_flags, stream_of(x)));
    if (inplace) {
        if (x.data_ptr() != input.data_ptr()) const_cast<at::Tensor&>(input).copy_(x);   // a non-contiguous input went through a copy
        return {meta, gamax, gnnz, gerr};
    }
    return {out, meta, gamax, gnnz, gerr};
}

at::Tensor e8mx_impl(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y, int64_t quantize_type,
                     int64_t scaling_strategy, const at::Tensor* result) {
    check_input(input, at::kBFloat16, dim_x, dim_y, "input");
    check_blocks(block_x, block_y);
    if (result) {
        check_input(*result, at::kBFloat16, dim_x, dim_y, "result");
        TORCH_CHECK(result->is_contiguous(), "mor: result must be contiguous");
    }
    const at::Tensor x = input.contiguous();
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor out = result ? *result : at::empty_like(x);
    const size_t nbytes = mor_workspace_bytes(MOR_OP_E8MX, dim_x, dim_y, block_x, block_y);
    at::Tensor ws = at::empty({(int64_t)nbytes}, x.options().dtype(at::kByte));
    check(mor_e8mx(x.data_ptr(), out.data_ptr(), dim_x, dim_y, block_x, block_y, quantize_type, scaling_strategy, ws.data_ptr(), nbytes,
                   g_flags, stream_of(x)));
    return out;
}

template <int FMT>
at::Tensor quant_dequant(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t, int64_t) {
    check_input(input, at::kFloat, dim_x, dim_y, "input");
    const at::Tensor x = input.contiguous();
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor out = at::empty_like(x);
    check(mor_quant_dequant(x.data_ptr<float>(), out.data_ptr<float>(), x.numel(), FMT, stream_of(x)));
    return out;
}

template <int RNE>
at::Tensor e8_scale(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t, int64_t) {
    check_input(input, at::kFloat, dim_x, dim_y, "input");
    const at::Tensor x = input.contiguous();
    const c10::OptionalDeviceGuard guard(x.device());
    at::Tensor out = at::empty_like(x);
    check(mor_e4m3_with_e8_scale(x.data_ptr<float>(), out.data_ptr<float>(), x.numel(), RNE, stream_of(x)));
    return out;
}

// Straight-through estimator (mor/ops.py:15-156): the gradient of the first output passes to the input unchanged.
// `call` runs the operator below the autograd key, through the dispatcher, so fake / functional tensors still trace.
using OpCall = std::function<std::vector<at::Tensor>(const at::Tensor&)>;
struct StraightThrough : public torch::autograd::Function<StraightThrough> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& input, OpCall call) {
        at::AutoDispatchBelowADInplaceOrView below;
        std::vector<at::Tensor> outs = call(input);
        if (outs.size() > 1) ctx->mark_non_differentiable(torch::autograd::variable_list(outs.begin() + 1, outs.end()));
        return outs;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list grads) {
        return {grads[0], at::Tensor()};
    }
};

std::vector<at::Tensor> fake_quantize_autograd(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y,
                                               double clamp_threshold, int64_t mode, int64_t sf_type) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("mor::fake_quantize", "")
        .typed<std::vector<at::Tensor>(const at::Tensor&, int64_t, int64_t, int64_t, int64_t, double, int64_t, int64_t)>();
    return StraightThrough::apply(input, OpCall([=](const at::Tensor& x) { return op.call(x, dim_x, dim_y, block_x, block_y, clamp_threshold, mode, sf_type); }));
}

template <bool CHANNEL>
std::vector<at::Tensor> scaling_autograd(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y,
                                         double e4m3_threshold, int64_t ss_mode) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow(CHANNEL ? "mor::fake_quantize_channel_scaling" : "mor::fake_quantize_block_scaling", "")
        .typed<std::vector<at::Tensor>(const at::Tensor&, int64_t, int64_t, int64_t, int64_t, double, int64_t)>();
    return StraightThrough::apply(input, OpCall([=](const at::Tensor& x) { return op.call(x, dim_x, dim_y, block_x, block_y, e4m3_threshold, ss_mode); }));
}

at::Tensor e8mx_autograd(const at::Tensor& input, int64_t dim_x, int64_t dim_y, int64_t block_x, int64_t block_y, int64_t quantize_type,
                         int64_t scaling_strategy) {
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("mor::fake_quantize_e8mx", "")
        .typed<at::Tensor(const at::Tensor&, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t)>();
    return StraightThrough::apply(input, OpCall([=](const at::Tensor& x) {
        return std::vector<at::Tensor>{op.call(x, dim_x, dim_y, block_x, block_y, quantize_type, scaling_strategy)}; }))[0];
}

// ---------------------------------------------------------------------------------------------------------------------
// The MX wire format and the operators on it (mor_amd/wire.py, mor_amd/mx.py; not in the reference)
int64_t payload_bytes(int64_t n, int64_t fmt) { return (int64_t)mor_mx_payload_bytes(1, n, (int)fmt); }

// contiguous and at a multiple of `bytes`: a view that is not is copied
at::Tensor aligned(const at::Tensor& t, uintptr_t bytes) {
    const at::Tensor x = t.contiguous();
    return reinterpret_cast<uintptr_t>(x.data_ptr()) % bytes ? x.clone() : x;
}

// A 2-D bf16 GPU tensor, contiguous and 16-byte aligned
at::Tensor wire_input(const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.is_cuda(), "mor: ", what, " must be a 2-D bfloat16 GPU tensor, got ",
                t.scalar_type(), " ", t.sizes());
    TORCH_CHECK(t.size(1) > 0 && t.size(1) % 32 == 0, "mor: ", what, ": MX blocks need columns that are a multiple of 32, got ", t.sizes());
    return aligned(t, 16);
}

std::tuple<at::Tensor, at::Tensor> mx_quantize(const at::Tensor& input, int64_t fmt) {
    const at::Tensor x = wire_input(input, "input");
    TORCH_CHECK(fmt >= MOR_FMT_E4M3 && fmt <= MOR_FMT_E2M1, "mor: unknown element format ", fmt);
    const c10::OptionalDeviceGuard guard(x.device());
    const auto u8 = x.options().dtype(at::kByte);
    const int64_t rows = x.size(0), cols = x.size(1);
    at::Tensor p = at::empty({rows, payload_bytes(cols, fmt)}, u8), s = at::empty({rows, cols / 32}, u8);
    if (rows) check(mor_mx_quantize(x.data_ptr(), p.data_ptr(), s.data_ptr(), rows, cols, (int)fmt, stream_of(x)));
    return {p, s};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> mx_quantize_dual(const at::Tensor& input, int64_t row_fmt, int64_t col_fmt) {
    const at::Tensor x = wire_input(input, "input");
    const c10::OptionalDeviceGuard guard(x.device());
    const auto u8 = x.options().dtype(at::kByte);
    const int64_t rows = x.size(0), cols = x.size(1), blocks = cdiv(rows, 32);
    at::Tensor rp = at::empty({rows, payload_bytes(cols, row_fmt)}, u8), rs = at::empty({rows, cols / 32}, u8);
    at::Tensor cp = at::empty({cols, rows ? payload_bytes(blocks * 32, col_fmt) : 0}, u8), cs = at::empty({cols, blocks}, u8);
    if (rows && row_fmt == col_fmt && rows % 32 == 0)
        check(mor_mx_quantize_dual(x.data_ptr(), rp.data_ptr(), rs.data_ptr(), cp.data_ptr(), cs.data_ptr(), rows, cols, (int)row_fmt, stream_of(x)));
    else if (rows) check(mor_mx_quantize_dual_ragged(x.data_ptr(), rp.data_ptr(), rs.data_ptr(), cp.data_ptr(), cs.data_ptr(), rows, cols,
                                                     (int)row_fmt, (int)col_fmt, stream_of(x)));
    return {rp, rs, cp, cs};
}

at::Tensor mx_dequantize(const at::Tensor& payload, const at::Tensor& scales, int64_t fmt) {
    TORCH_CHECK(payload.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && payload.is_cuda() && payload.device() == scales.device() && scales.dim() == 2,
                "mor: expected uint8 GPU tensors");
    TORCH_CHECK(fmt >= MOR_FMT_E4M3 && fmt <= MOR_FMT_E2M1, "mor: unknown element format ", fmt);
    const int64_t rows = scales.size(0), cols = scales.size(1) * 32;
    TORCH_CHECK(payload.numel() == (cols ? rows * payload_bytes(cols, fmt) : 0), "mor: payload size does not match the scales");
    const at::Tensor p = aligned(payload, 16), s = aligned(scales, 4);
    const c10::OptionalDeviceGuard guard(p.device());
    at::Tensor out = at::empty({rows, cols}, p.options().dtype(at::kBFloat16));
    if (rows) check(mor_mx_dequantize(p.data_ptr(), s.data_ptr(), out.data_ptr(), rows, cols, (int)fmt, stream_of(p)));
    return out;
}

at::Tensor mx_matmul(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& b, const at::Tensor& b_scales, int64_t a_fmt, int64_t b_fmt) {
    auto side = [](const at::Tensor& p, const at::Tensor& s, int64_t fmt, const char* what) {
        TORCH_CHECK(p.scalar_type() == at::kByte && s.scalar_type() == at::kByte && p.is_cuda() && p.device() == s.device() && p.dim() == 2 && s.dim() == 2,
                    "mor: ", what, ": expected a 2-D uint8 payload and 2-D uint8 scales on one GPU");
        TORCH_CHECK(fmt == MOR_FMT_E4M3 || fmt == MOR_FMT_E5M2 || fmt == MOR_FMT_E2M1, "mor: ", what, ": products take the formats E4M3, E5M2 and E2M1, got ", fmt);
        TORCH_CHECK(p.size(0) == s.size(0) && p.size(1) == s.size(1) * (fmt == MOR_FMT_E2M1 ? 16 : 32), "mor: ", what, ": payload ", p.sizes(),
                    " does not match scales ", s.sizes());
    };
    side(a, a_scales, a_fmt, "a");
    side(b, b_scales, b_fmt, "b");
    TORCH_CHECK(a.device() == b.device(), "mor: a and b must be on one device");
    TORCH_CHECK(a_scales.size(1) == b_scales.size(1), "mor: a and b must have the same number of columns, got ", a_scales.size(1) * 32, " and ", b_scales.size(1) * 32);
    const at::Tensor pa = aligned(a, 16), sa = a_scales.contiguous(), pb = aligned(b, 16), sb = b_scales.contiguous();
    const c10::OptionalDeviceGuard guard(pa.device());
    const int64_t m = pa.size(0), n = pb.size(0), k = sa.size(1) * 32;
    const auto options = pa.options().dtype(at::kBFloat16);
    if (k == 0) return at::zeros({m, n}, options);
    at::Tensor out = at::empty({m, n}, options);
    if (m == 0 || n == 0) return out;
    const size_t nbytes = mor_mx_matmul_workspace_bytes(m, n, k, (int)a_fmt, (int)b_fmt);
    at::Tensor ws;
    if (nbytes) ws = at::empty({(int64_t)nbytes}, pa.options());
    check(mor_mx_matmul(pa.data_ptr(), sa.data_ptr(), (int)a_fmt, pb.data_ptr(), sb.data_ptr(), (int)b_fmt, out.data_ptr(), m, n, k,
                        nbytes ? ws.data_ptr() : nullptr, nbytes, stream_of(pa)));
    return out;
}

// rows of contiguous elements at one stride, as they lie; anything else is copied
at::Tensor rows_of(const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.is_cuda(), "mor: ", what, " must be a 2-D bfloat16 GPU tensor, got ",
                t.scalar_type(), " ", t.sizes());
    const bool as_is = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return as_is ? t : t.contiguous();
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// The 8-bit copies of gate and up in one buffer: codes of gate, of up, scale bytes of gate, of up
struct SwigluKept {
    int64_t codes, scales, bytes;
    SwigluKept(int64_t rows, int64_t cols) : codes((rows * cdiv(cols, 32) * 32 + 255) / 256 * 256), scales(rows * cdiv(cols, 32)), bytes(2 * (codes + scales)) {}
};

std::tuple<at::Tensor, at::Tensor> swiglu_forward(const at::Tensor& gate, const at::Tensor& up, bool keep) {
    const at::Tensor g = rows_of(gate, "gate"), u = rows_of(up, "up");
    TORCH_CHECK(g.sizes() == u.sizes() && g.device() == u.device(), "mor: gate and up must have the same shape and device, got ", g.sizes(), " and ", u.sizes());
    const c10::OptionalDeviceGuard guard(g.device());
    const int64_t rows = g.size(0), cols = g.size(1);
    at::Tensor out = at::empty({rows, cols}, g.options());
    const SwigluKept k(rows, cols);
    at::Tensor kept = at::empty({keep ? k.bytes : 0}, g.options().dtype(at::kByte));
    uint8_t* b = keep ? kept.data_ptr<uint8_t>() : nullptr;
    if (out.numel()) check(mor_swiglu_mx(g.data_ptr(), row_stride(g), u.data_ptr(), row_stride(u), out.data_ptr(), b, b ? b + 2 * k.codes : nullptr,
                                         b ? b + k.codes : nullptr, b ? b + 2 * k.codes + k.scales : nullptr, rows, cols, stream_of(g)));
    return {out, kept};
}

std::tuple<at::Tensor, at::Tensor> swiglu_backward(const at::Tensor& grad, const at::Tensor& kept) {
    TORCH_CHECK(grad.scalar_type() == at::kBFloat16 && grad.dim() == 2 && grad.is_cuda(), "mor: grad must be a 2-D bfloat16 GPU tensor, got ", grad.scalar_type(), " ", grad.sizes());
    const at::Tensor d = grad.contiguous();
    const int64_t rows = d.size(0), cols = d.size(1);
    const SwigluKept k(rows, cols);
    TORCH_CHECK(kept.scalar_type() == at::kByte && kept.device() == d.device() && kept.is_contiguous() && kept.numel() == k.bytes, "mor: kept does not match grad");
    const at::Tensor at16 = aligned(kept, 16);             // (a saved-tensor hook may bring it back anywhere)
    const c10::OptionalDeviceGuard guard(d.device());
    at::Tensor dg = at::empty({rows, cols}, d.options()), du = at::empty({rows, cols}, d.options());
    const uint8_t* b = at16.data_ptr<uint8_t>();
    if (d.numel()) check(mor_swiglu_mx_backward(d.data_ptr(), b, b + 2 * k.codes, b + k.codes, b + 2 * k.codes + k.scales, dg.data_ptr(), du.data_ptr(), rows, cols, stream_of(d)));
    return {dg, du};
}

// The linear layer.  Its codes lie in one buffer per lifetime (an allocation costs as much host time as a launch): those
// of the forward product, those that the backward pass needs, those of dy.
struct Parts {
    int64_t bytes = 0;
    int64_t add(int64_t n) { const int64_t at = bytes; bytes += (n + 255) / 256 * 256; return at; }
};
struct Codes { uint8_t *payload, *scales; };
struct CodesAt {
    int64_t payload, scales;
    static CodesAt in(Parts& p, int64_t rows, int64_t cols, int64_t fmt) {
        const int64_t a = p.add(rows && cols ? rows * payload_bytes(cols, fmt) : 0);
        return {a, p.add(rows * (cols / 32))};
    }
    Codes of(const at::Tensor& buffer) const { uint8_t* b = buffer.data_ptr<uint8_t>(); return {b + payload, b + scales}; }
};
struct Kept {          // x^T [inputs, tokens filled up to blocks] in E4M3 and weight^T [inputs, outputs] in fmt
    Parts parts;
    CodesAt xt{}, wt{};
    Kept(int64_t tokens, int64_t inputs, int64_t outputs, int64_t fmt, bool keep_x, bool keep_w) {
        if (keep_x) xt = CodesAt::in(parts, inputs, cdiv(tokens, 32) * 32, MOR_FMT_E4M3);
        if (keep_w) wt = CodesAt::in(parts, inputs, outputs, fmt);
    }
};

void quantize_into(const at::Tensor& x, int64_t fmt, Codes rows) {
    check(mor_mx_quantize(x.data_ptr(), rows.payload, rows.scales, x.size(0), x.size(1), (int)fmt, stream_of(x)));
}
void quantize_into(const at::Tensor& x, int64_t row_fmt, Codes rows, int64_t col_fmt, Codes cols) {
    check(mor_mx_quantize_dual_ragged(x.data_ptr(), rows.payload, rows.scales, cols.payload, cols.scales, x.size(0), x.size(1), (int)row_fmt, (int)col_fmt, stream_of(x)));
}
at::Tensor product(Codes a, int64_t a_fmt, Codes b, int64_t b_fmt, int64_t m, int64_t n, int64_t k, const at::TensorOptions& options, void* stream) {
    at::Tensor out = at::empty({m, n}, options.dtype(at::kBFloat16)), ws;
    const size_t nbytes = mor_mx_matmul_workspace_bytes(m, n, k, (int)a_fmt, (int)b_fmt);
    if (nbytes) ws = at::empty({(int64_t)nbytes}, options.dtype(at::kByte));
    check(mor_mx_matmul(a.payload, a.scales, (int)a_fmt, b.payload, b.scales, (int)b_fmt, out.data_ptr(), m, n, k, nbytes ? ws.data_ptr() : nullptr, nbytes, stream));
    return out;
}

void check_linear(const at::Tensor& x, const at::Tensor& w, int64_t fmt) {
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.is_cuda() && x.dim() == 2, "mor: x must be a bfloat16 GPU tensor, got ", x.scalar_type());
    TORCH_CHECK(w.scalar_type() == at::kBFloat16 && w.device() == x.device() && w.dim() == 2, "mor: weight must be a 2-D bfloat16 tensor on the device of x, got ",
                w.scalar_type(), " ", w.sizes());
    TORCH_CHECK(x.size(1) == w.size(1), "mor: x has ", x.size(1), " columns, weight has ", w.size(1));
    TORCH_CHECK(w.size(0) > 0 && w.size(0) % 32 == 0 && w.size(1) > 0 && w.size(1) % 32 == 0, "mor: inputs and outputs must be multiples of 32, got weight ", w.sizes());
    TORCH_CHECK(fmt == MOR_FMT_E4M3 || fmt == MOR_FMT_E2M1, "mor: fmt must be E4M3 or E2M1, got ", fmt);
}
void check_grad_fmt(int64_t grad_fmt) { TORCH_CHECK(grad_fmt == MOR_FMT_E4M3 || grad_fmt == MOR_FMT_E5M2, "mor: grad_fmt must be E4M3 or E5M2, got ", grad_fmt); }

// y = Q(x) Q(w)^T, and what the backward pass needs: x^T if the weight wants a gradient, weight^T if x does
std::tuple<at::Tensor, at::Tensor> linear_forward(const at::Tensor& input, const at::Tensor& weight, int64_t fmt, bool keep_x, bool keep_w) {
    check_linear(input, weight, fmt);
    const at::Tensor x = wire_input(input, "x"), w = wire_input(weight, "weight");
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t tokens = x.size(0), inputs = x.size(1), outputs = w.size(0);
    // (each of them is the summed axis of a product: refused here rather than in the backward pass)
    TORCH_CHECK((!keep_x || tokens <= (1 << 23) - 32) && inputs < (1 << 23) && outputs < (1 << 23),
                "mor: at most 2^23 - 32 tokens, inputs and outputs, got ", tokens, ", ", inputs, " and ", outputs);
    const auto u8 = x.options().dtype(at::kByte);
    Parts scratch;
    const CodesAt xr = CodesAt::in(scratch, tokens, inputs, fmt), wr = CodesAt::in(scratch, outputs, inputs, fmt);
    const Kept k(tokens, inputs, outputs, fmt, keep_x, keep_w);
    const at::Tensor rows = at::empty({scratch.bytes}, u8);
    at::Tensor kept = at::empty({k.parts.bytes}, u8);
    if (keep_w) quantize_into(w, fmt, wr.of(rows), fmt, k.wt.of(kept));
    else quantize_into(w, fmt, wr.of(rows));
    if (tokens == 0) return {at::empty({0, outputs}, x.options()), kept};
    if (keep_x) quantize_into(x, fmt, xr.of(rows), MOR_FMT_E4M3, k.xt.of(kept));
    else quantize_into(x, fmt, xr.of(rows));
    return {product(xr.of(rows), fmt, wr.of(rows), fmt, tokens, outputs, inputs, u8, stream_of(x)), kept};
}

std::tuple<at::Tensor, at::Tensor> linear_backward(const at::Tensor& grad, const at::Tensor& kept, int64_t inputs, int64_t fmt, int64_t grad_fmt, bool kept_x, bool kept_w) {
    check_grad_fmt(grad_fmt);
    const at::Tensor d = wire_input(grad, "grad");
    const int64_t tokens = d.size(0), outputs = d.size(1), padded = cdiv(tokens, 32) * 32;
    const Kept k(tokens, inputs, outputs, fmt, kept_x, kept_w);
    TORCH_CHECK(kept.scalar_type() == at::kByte && kept.device() == d.device() && kept.is_contiguous() && kept.numel() == k.parts.bytes, "mor: kept does not match grad");
    const at::Tensor at16 = aligned(kept, 16);             // (a saved-tensor hook may bring it back anywhere)
    const c10::OptionalDeviceGuard guard(d.device());
    const auto u8 = d.options().dtype(at::kByte);
    at::Tensor dx = at::empty({0}, d.options()), dw = dx;
    if (tokens == 0) {
        if (kept_w) dx = at::empty({0, inputs}, d.options());
        if (kept_x) dw = at::zeros({outputs, inputs}, d.options());
        return {dx, dw};
    }
    Parts scratch;
    const CodesAt gr = CodesAt::in(scratch, tokens, outputs, grad_fmt), gt = kept_x ? CodesAt::in(scratch, outputs, padded, grad_fmt) : CodesAt{};
    const at::Tensor codes = at::empty({scratch.bytes}, u8);
    if (kept_x) quantize_into(d, grad_fmt, gr.of(codes), grad_fmt, gt.of(codes));
    else quantize_into(d, grad_fmt, gr.of(codes));
    if (kept_w) dx = product(gr.of(codes), grad_fmt, k.wt.of(at16), fmt, tokens, inputs, outputs, u8, stream_of(d));
    if (kept_x) dw = product(gt.of(codes), grad_fmt, k.xt.of(at16), MOR_FMT_E4M3, outputs, inputs, padded, u8, stream_of(d));
    return {dx, dw};
}

// the operators above through the dispatcher, so that fake tensors trace
template <class Sig> c10::TypedOperatorHandle<Sig> handle(const char* name) { return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>(); }
std::tuple<at::Tensor, at::Tensor> call_linear(const at::Tensor& x, const at::Tensor& w, int64_t fmt, bool keep_x, bool keep_w) {
    static auto op = handle<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, int64_t, bool, bool)>("mor::mx_linear_forward");
    return op.call(x, w, fmt, keep_x, keep_w);
}
at::Tensor mx_linear(const at::Tensor& x, const at::Tensor& w, int64_t fmt, int64_t grad_fmt) {
    check_grad_fmt(grad_fmt);
    return std::get<0>(call_linear(x, w, fmt, false, false));
}

// A leaf's gradient is added on the stream that its live graphs were built on.  Where one was built on the default stream,
// a backward pass under capture would have that stream wait for the captured one, which cannot be captured and ends the
// process: refused while nothing is captured yet.  (Graphs built on another stream join the capture and leave it again.)
void check_capture(const at::Tensor& a, const at::Tensor& b) {
    const int device = a.device().index();
    if (!a.is_cuda() || a.key_set().has(c10::DispatchKey::Python)) return;                       // (fake tensors)
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device).stream(), &status) != hipSuccess) {
        (void)hipGetLastError();
        return;
    }
    if (status == hipStreamCaptureStatusNone) return;
    for (const at::Tensor& t : {a, b}) {
        if (!t.requires_grad()) continue;
        std::shared_ptr<torch::autograd::Node> node = t.grad_fn();
        if (!node) node = torch::autograd::impl::try_get_grad_accumulator(t);
        while (node && node->num_outputs() == 1) node = node->next_edge(0).function;             // views of a leaf
        if (!node || !dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(device).id(),
                    "mor: a graph built on the default stream holds a leaf of this call, whose backward pass cannot be captured then; "
                    "free that graph first, build it on a side stream, or, for a forward pass alone, call under torch.no_grad()");
    }
}

// A tangent would be lost without a word: below the autograd key nothing carries one (torch.func.jvp, forward_ad; a dual
// tensor need not require a gradient).
void refuse_tangents(std::initializer_list<at::Tensor> inputs, const char* what) {
    for (const at::Tensor& t : inputs)
        TORCH_CHECK(!(t.defined() && t._fw_grad(0).defined()), "mor: ", what, " has no forward-mode derivative");
}

// The quantisers are passed straight through.
struct MxLinear : public torch::autograd::Function<MxLinear> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, int64_t fmt, int64_t grad_fmt,
                              bool need_x, bool need_w) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, kept] = call_linear(x, w, fmt, need_w, need_x);
        ctx->save_for_backward({kept});
        ctx->saved_data["call"] = w.size(1) << 8 | fmt << 4 | grad_fmt << 2 | (int64_t)need_w << 1 | (int64_t)need_x;      // (fmt 0 or 4, grad_fmt 0 or 1)
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "mor: mx.linear has no second derivative");
        refuse_tangents({grads[0]}, "the gradient of mx.linear");
        at::Tensor dx, dw;
        if (grads[0].defined()) {
            static auto op = handle<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, int64_t, int64_t, int64_t, bool, bool)>("mor::mx_linear_backward");
            const int64_t call = ctx->saved_data["call"].toInt();
            const bool need_w = call & 2, need_x = call & 1;
            std::tie(dx, dw) = op.call(grads[0], ctx->get_saved_variables()[0], call >> 8, call >> 4 & 15, call >> 2 & 3, need_w, need_x);
            if (!need_x) dx = at::Tensor();
            if (!need_w) dw = at::Tensor();
        }
        return {dx, dw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

at::Tensor mx_linear_autograd(const at::Tensor& x, const at::Tensor& w, int64_t fmt, int64_t grad_fmt) {
    check_grad_fmt(grad_fmt);
    refuse_tangents({x, w}, "mx.linear");
    const bool on = at::GradMode::is_enabled(), need_x = on && x.requires_grad(), need_w = on && w.requires_grad();
    if (!need_x && !need_w) {
        at::AutoDispatchBelowADInplaceOrView below;
        return std::get<0>(call_linear(x, w, fmt, false, false));
    }
    check_capture(x, w);
    return MxLinear::apply(x, w, fmt, grad_fmt, need_x, need_w);
}

std::tuple<at::Tensor, at::Tensor> call_swiglu(const at::Tensor& gate, const at::Tensor& up, bool keep) {
    static auto op = handle<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&, bool)>("mor::swiglu_mx_forward");
    return op.call(gate, up, keep);
}
struct SwigluMx : public torch::autograd::Function<SwigluMx> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& gate, const at::Tensor& up) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [h, kept] = call_swiglu(gate, up, true);
        ctx->save_for_backward({kept});
        return h;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "mor: mx.swiglu has no second derivative");
        refuse_tangents({grads[0]}, "the gradient of mx.swiglu");
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
        static auto op = handle<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const at::Tensor&)>("mor::swiglu_mx_backward");
        auto [dg, du] = op.call(grads[0], ctx->get_saved_variables()[0]);
        return {dg, du};
    }
};
at::Tensor swiglu(const at::Tensor& gate, const at::Tensor& up) { return std::get<0>(call_swiglu(gate, up, false)); }
at::Tensor swiglu_autograd(const at::Tensor& gate, const at::Tensor& up) {
    refuse_tangents({gate, up}, "mx.swiglu");
    if (!at::GradMode::is_enabled() || !(gate.requires_grad() || up.requires_grad())) {
        at::AutoDispatchBelowADInplaceOrView below;
        return std::get<0>(call_swiglu(gate, up, false));
    }
    check_capture(gate, up);
    return SwigluMx::apply(gate, up);
}

}  // namespace

// mor.ops.set_flavour: MOR_FLAG_* bits for every later call of the calling thread
extern "C" __attribute__((visibility("default"))) void mor_torch_set_flags(uint32_t flags) { g_flags = flags; }

static void mx_operators(torch::Library& m) {
    m.impl("mx_quantize", &mx_quantize);
    m.impl("mx_quantize_dual", &mx_quantize_dual);
    m.impl("mx_dequantize", &mx_dequantize);
    m.impl("mx_matmul", &mx_matmul);
    m.impl("mx_linear", &mx_linear);
    m.impl("mx_linear_forward", &linear_forward);
    m.impl("mx_linear_backward", &linear_backward);
    m.impl("swiglu_mx", &swiglu);
    m.impl("swiglu_mx_forward", &swiglu_forward);
    m.impl("swiglu_mx_backward", &swiglu_backward);
}

TORCH_LIBRARY_IMPL(mor, CUDA, m) {
    m.impl("fake_quantize", &fake_quantize);
    m.impl("fake_quantize_no_alloc", &fake_quantize_no_alloc);
    m.impl("quant_dequant_e4m3", &quant_dequant<MOR_FMT_E4M3>);
    m.impl("quant_dequant_e5m2", &quant_dequant<MOR_FMT_E5M2>);
    m.impl("quant_dequant_e3m2", &quant_dequant<MOR_FMT_E3M2>);
    m.impl("quant_dequant_e2m3", &quant_dequant<MOR_FMT_E2M3>);
    m.impl("e4m3_with_e8_scale_rne", &e8_scale<1>);
    m.impl("e4m3_with_e8_scale_rz", &e8_scale<0>);
    m.impl("fake_quantize_block_scaling", [](const at::Tensor& i, int64_t x, int64_t y, int64_t bx, int64_t by, double t, int64_t s) {
        return scaling(i, x, y, bx, by, t, s, false, false); });
    m.impl("fake_quantize_block_scaling_inplace", [](const at::Tensor& i, int64_t x, int64_t y, int64_t bx, int64_t by, double t, int64_t s) {
        return scaling(i, x, y, bx, by, t, s, false, true); });
    m.impl("fake_quantize_channel_scaling", [](const at::Tensor& i, int64_t x, int64_t y, int64_t bx, int64_t by, double t, int64_t s) {
        return scaling(i, x, y, bx, by, t, s, true, false); });
    m.impl("fake_quantize_channel_scaling_inplace", [](const at::Tensor& i, int64_t x, int64_t y, int64_t bx, int64_t by, double t, int64_t s) {
        return scaling(i, x, y, bx, by, t, s, true, true); });
    m.impl("fake_quantize_e8mx", [](const at::Tensor& i, int64_t x, int64_t y, int64_t bx, int64_t by, int64_t q, int64_t s) {
        return e8mx_impl(i, x, y, bx, by, q, s, nullptr); });
    m.impl("fake_quantize_e8mx_inplace", [](const at::Tensor& i, int64_t x, int64_t y, int64_t bx, int64_t by, int64_t q, int64_t s, at::Tensor result) {
        e8mx_impl(i, x, y, bx, by, q, s, &result); });
    mx_operators(m);
}

// (tensors in host memory: their checks refuse them by name)
TORCH_LIBRARY_IMPL(mor, CPU, m) { mx_operators(m); }

// autograd for the four differentiable forward ops; the in-place / no_alloc / test ops keep their Python registration
TORCH_LIBRARY_IMPL(mor, Autograd, m) {
    m.impl("fake_quantize", &fake_quantize_autograd);
    m.impl("fake_quantize_block_scaling", &scaling_autograd<false>);
    m.impl("fake_quantize_channel_scaling", &scaling_autograd<true>);
    m.impl("fake_quantize_e8mx", &e8mx_autograd);
    m.impl("mx_linear", &mx_linear_autograd);
    m.impl("swiglu_mx", &swiglu_autograd);
}
