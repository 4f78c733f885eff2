// Microscaled (MX) operators, registered next to the reference's: a decoder's linears on 4-bit
// weights with 8- or 4-bit activations. The reference has no counterpart (its tensors are fp32).
//
//   mx_quantize     x -> codes, scales
//   mx_dequantize   codes, scales -> values
//   rms_norm_mx     rms_norm (with the residual add before it) -> codes, scales
//   silu_mul_mx     act_fn and mul of the MLP -> codes, scales
//   mx_linear       x codes, x scales, weight codes, weight scales (, bias) (, residual) -> out
//
// codes and scales are uint8 tensors whose last dimensions tell the format: scales [.., K / 32];
// codes [.., K] for e4m3 ("fp8"), [.., K / 2] for e2m1 ("fp4").
#include "common.h"

namespace dli::plugin {
namespace {

std::int64_t rowsOf(const Tensor& t) { return product(t.shape(), 0, t.rank() - 1); }

// Every input is on the device that the call's launches go to.
void requireOneDevice(const std::vector<const Tensor*>& in, const std::string& op) {
  requireCudaInputs(in, op);
  int current = 0;
  check(dli_hip_get_device(&current), op);
  for (const Tensor* t : in)
    if (t->deviceId() != current)
      throw std::invalid_argument(op + " expects its tensors on the current device");
}

int formatAttr(const Attributes& attrs, const std::string& op) {
  const std::string format = attrs.value_or<std::string>("format", "fp8");
  if (format == "fp8") return DLI_MX_FP8;
  if (format == "fp4") return DLI_MX_FP4;
  throw std::invalid_argument(op + " format must be fp8 or fp4, not " + format);
}

// Allocates codes and scales for rows of `width` values, leading dimensions as in `shape`.
void allocate(std::vector<std::int64_t> shape, std::int64_t width, int format, int device_id,
              const std::string& op, Tensor& codes, Tensor& scales) {
  if (width <= 0 || width % 32 != 0)
    throw std::invalid_argument(op + ": the last dimension must be a positive multiple of 32");
  codes = Tensor::cuda(DType::UInt8, withLast(shape, format == DLI_MX_FP8 ? width : width / 2),
                       device_id);
  scales = Tensor::cuda(DType::UInt8, withLast(shape, width / 32), device_id);
}

// Format and width of a microscaled tensor from its two shapes.
int formatOf(const Tensor& codes, const Tensor& scales, const std::string& op,
             const std::string& what, std::int64_t* width) {
  if (codes.dtype() != DType::UInt8 || scales.dtype() != DType::UInt8)
    throw std::invalid_argument(op + " " + what + " codes and scales must be uint8");
  const std::int64_t s = scales.shape().back(), c = codes.shape().back();
  if (codes.rank() != scales.rank() || s <= 0 || (c != s * 32 && c != s * 16))
    throw std::invalid_argument(op + " " + what + ": codes " + formatShape(codes.shape()) +
                                " and scales " + formatShape(scales.shape()) +
                                " are not a microscaled tensor");
  for (std::size_t i = 0; i + 1 < codes.rank(); ++i)
    if (codes.dim(i) != scales.dim(i))
      throw std::invalid_argument(op + " " + what + ": codes and scales have different rows");
  *width = s * 32;
  return c == s * 32 ? DLI_MX_FP8 : DLI_MX_FP4;
}

// inputs: x [.., K]; attr format ("fp8", "fp4"); outputs: codes, scales
class MxQuantizeOp final : public Operator {
 public:
  std::string type() const override { return "mx_quantize"; }
  void compute(const std::vector<const Tensor*>& in, const std::vector<Tensor*>& out,
               const Attributes& attrs, ExecutionContext& ctx) const override {
    requireArity(in, out, 1, 1, 2, type());
    requireOneDevice(in, type());
    const Tensor& x = *in[0];
    requireFloating(x, type());
    const int format = formatAttr(attrs, type());
    const std::int64_t k = x.shape().back();
    allocate(x.shape(), k, format, x.deviceId(), type(), *out[0], *out[1]);
    check(dli_hip_mx_quantize(hipDtype(x.dtype()), format, ptr(x), ptr(*out[0]), ptr(*out[1]),
                              rowsOf(x), k, ctx.stream),
          type());
  }
};

// inputs: codes, scales; attr dtype ("bfloat16", "float16", "float32"); output: values [.., K]
class MxDequantizeOp final : public Operator {
 public:
  std::string type() const override { return "mx_dequantize"; }
  void compute(const std::vector<const Tensor*>& in, const std::vector<Tensor*>& out,
               const Attributes& attrs, ExecutionContext& ctx) const override {
    requireArity(in, out, 2, 2, 1, type());
    requireOneDevice(in, type());
    std::int64_t k = 0;
    const int format = formatOf(*in[0], *in[1], type(), "input", &k);
    const DType dtype = dtypeFromString(attrs.value_or<std::string>("dtype", "bfloat16"));
    if (!isFloating(dtype)) throw std::invalid_argument(type() + " dtype must be a floating type");
    *out[0] = Tensor::cuda(dtype, withLast(in[0]->shape(), k), in[0]->deviceId());
    check(dli_hip_mx_dequantize(hipDtype(dtype), format, ptr(*in[0]), ptr(*in[1]), ptr(*out[0]),
                                rowsOf(*in[0]), k, ctx.stream),
          type());
  }
};

// inputs: x [.., H], weight [H] (, residual [.., H]); attrs eps, format; outputs: codes, scales
// and, with a residual, hidden = x + residual
class RmsNormMxOp final : public Operator {
 public:
  std::string type() const override { return "rms_norm_mx"; }
  void compute(const std::vector<const Tensor*>& in, const std::vector<Tensor*>& out,
               const Attributes& attrs, ExecutionContext& ctx) const override {
    requireArity(in, out, 2, 3, in.size() == 3 ? 3 : 2, type());
    requireOneDevice(in, type());
    const Tensor &x = *in[0], &w = *in[1];
    const Tensor* residual = in.size() == 3 ? in[2] : nullptr;
    requireFloating(x, type());
    requireSameDType(x, w, type());
    const std::int64_t hidden = x.shape().back();
    if (static_cast<std::int64_t>(w.numel()) != hidden)
      throw std::invalid_argument("rms_norm_mx weight size must match the last input dim");
    if (residual != nullptr) {
      requireSameDType(x, *residual, type());
      if (!sameShape(x, *residual))
        throw std::invalid_argument("rms_norm_mx residual must have the shape of x");
    }
    const int format = formatAttr(attrs, type());
    const auto eps = static_cast<float>(attrDouble(attrs, "eps", 1e-6));
    allocate(x.shape(), hidden, format, x.deviceId(), type(), *out[0], *out[1]);
    if (residual != nullptr) *out[2] = Tensor::cuda(x.dtype(), x.shape(), x.deviceId());
    check(dli_hip_rms_norm_mx(hipDtype(x.dtype()), format, ptr(x),
                              residual ? ptr(*residual) : nullptr, ptr(w),
                              residual ? ptr(*out[2]) : nullptr, ptr(*out[0]), ptr(*out[1]),
                              rowsOf(x), hidden, eps, ctx.stream),
          type());
  }
};

// inputs: gate, up [.., F], or one tensor [.., 2F] with gate in the first half of each row; attr
// format; outputs: codes, scales
class SiluMulMxOp final : public Operator {
 public:
  std::string type() const override { return "silu_mul_mx"; }
  void compute(const std::vector<const Tensor*>& in, const std::vector<Tensor*>& out,
               const Attributes& attrs, ExecutionContext& ctx) const override {
    requireArity(in, out, 1, 2, 2, type());
    requireOneDevice(in, type());
    const Tensor& gate = *in[0];
    requireFloating(gate, type());
    const std::int64_t stride = gate.shape().back();
    std::int64_t ffn = stride;
    const void* up = nullptr;
    if (in.size() == 2) {
      requireSameDType(gate, *in[1], type());
      if (!sameShape(gate, *in[1]))
        throw std::invalid_argument("silu_mul_mx gate and up must have one shape");
      up = ptr(*in[1]);
    } else {
      if (stride % 2 != 0)
        throw std::invalid_argument("silu_mul_mx: a joined gate and up has an even last dimension");
      ffn = stride / 2;
    }
    const int format = formatAttr(attrs, type());
    allocate(gate.shape(), ffn, format, gate.deviceId(), type(), *out[0], *out[1]);
    if (up == nullptr)
      up = static_cast<const char*>(ptr(gate)) + ffn * static_cast<std::int64_t>(byteSize(gate.dtype()));
    check(dli_hip_silu_mul_mx(hipDtype(gate.dtype()), format, ptr(gate), up, stride, ptr(*out[0]),
                              ptr(*out[1]), rowsOf(gate), ffn, ctx.stream),
          type());
  }
};

// inputs: x codes, x scales [.., K], weight codes, weight scales [N, K] (fp4) (, bias [N])
// (, residual [.., N]); attrs out_dtype ("bfloat16", "float16", "float32"), residual (whether the
// last input is one; an input between is the bias). bias and residual are of out_dtype.
class MxLinearOp final : public Operator {
 public:
  std::string type() const override { return "mx_linear"; }
  void compute(const std::vector<const Tensor*>& in, const std::vector<Tensor*>& out,
               const Attributes& attrs, ExecutionContext& ctx) const override {
    const bool has_residual = attrs.value_or<bool>("residual", false);
    requireArity(in, out, has_residual ? 5 : 4, has_residual ? 6 : 5, 1, type());
    requireOneDevice(in, type());
    const Tensor &x = *in[0], &w = *in[2];
    std::int64_t k = 0, wk = 0;
    const int x_format = formatOf(x, *in[1], type(), "x", &k);
    if (w.rank() != 2) throw std::invalid_argument("mx_linear weight must be 2-D");
    if (formatOf(w, *in[3], type(), "weight", &wk) != DLI_MX_FP4)
      throw std::invalid_argument("mx_linear weight must be fp4");
    if (k != wk)
      throw std::invalid_argument("mx_linear weight shape " + formatShape(w.shape()) +
                                  " does not match input " + formatShape(x.shape()));
    const std::int64_t n = w.dim(0), m = rowsOf(x);
    const DType dtype = dtypeFromString(attrs.value_or<std::string>("out_dtype", "bfloat16"));
    if (!isFloating(dtype)) throw std::invalid_argument("mx_linear out_dtype must be a floating type");
    const Tensor* bias = in.size() == (has_residual ? 6u : 5u) ? in[4] : nullptr;
    const Tensor* residual = has_residual ? in.back() : nullptr;
    if (bias != nullptr &&
        (bias->dtype() != dtype || static_cast<std::int64_t>(bias->numel()) != n))
      throw std::invalid_argument("mx_linear bias must have the output features and out_dtype");
    const std::vector<std::int64_t> shape = withLast(x.shape(), n);
    if (residual != nullptr && (residual->dtype() != dtype || residual->shape() != shape))
      throw std::invalid_argument("mx_linear residual must have the output's shape and out_dtype");
    *out[0] = Tensor::cuda(dtype, shape, x.deviceId());
    CallScratch scratch(dli_hip_mx_linear_workspace(x_format, m, n, k), x.deviceId());
    check(dli_hip_mx_linear(x_format, hipDtype(dtype), ptr(x), ptr(*in[1]), ptr(w), ptr(*in[3]),
                            bias ? ptr(*bias) : nullptr, residual ? ptr(*residual) : nullptr,
                            ptr(*out[0]), m, n, k, scratch.data(), scratch.bytes(), ctx.stream),
          type());
  }
};

}  // namespace

void registerMxOps(OperatorRegistry* registry) {
  add<MxQuantizeOp>(registry);
  add<MxDequantizeOp>(registry);
  add<RmsNormMxOp>(registry);
  add<SiluMulMxOp>(registry);
  add<MxLinearOp>(registry);
}

}  // namespace dli::plugin
