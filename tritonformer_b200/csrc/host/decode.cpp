// Weights in 4 bits and drawing tokens above the C ABI: checks, allocation and launch.  These operators have no gradients.
#include <cmath>

#include "functions.h"

namespace tfb_host {

static bool is_16_bit(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

Int4 int4_quantize(const Tensor& weight, int64_t group) {
  check_plain("quantize_int4", {&weight});
  BodyGuard guard;
  TFB_ASSERT(weight.defined() && weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0 && is_16_bit(weight.scalar_type()),
             "quantize_int4 expects an fp16/bf16 weight (in, out)");
  TFB_ASSERT(group == 32 || group == 64 || group == 128, "the groups are of 32, 64 or 128 rows");
  const c10::cuda::CUDAGuard device(weight.device());
  Int4 q;
  q.in = weight.size(0);
  q.out = weight.size(1);
  q.group = group;
  const int64_t strips = (q.out + 15) / 16;
  q.codes = at::empty({strips, (q.in + 63) / 64, 32, 4}, weight.options().dtype(at::kInt));
  q.scales = at::empty({strips, tfb_int4_scales(q.in, 1, (int)group) / 16, 8, 2}, weight.options());
  check(tfb_int4_quantize(weight.data_ptr(), weight.stride(0), weight.stride(1), q.in, q.out, (int)group, q.codes.data_ptr(),
                          q.scales.data_ptr(), dtype_code(weight.scalar_type()), current_stream(weight)));
  return q;
}

static void check_int4(const Int4& w) {
  TFB_ASSERT(w.in > 0 && w.out > 0 && w.in < (1 << 30) && w.out < (1 << 30), "a packed weight has rows and columns");
  TFB_ASSERT(w.group == 32 || w.group == 64 || w.group == 128, "the groups are of 32, 64 or 128 rows");
  TFB_ASSERT(w.codes.defined() && w.codes.scalar_type() == at::kInt && w.codes.is_contiguous() &&
                 w.codes.numel() == tfb_int4_codes(w.in, w.out),
             "the codes of a packed weight are those of quantize_int4");
  TFB_ASSERT(w.scales.defined() && is_16_bit(w.scales.scalar_type()) && w.scales.is_contiguous() &&
                 w.scales.numel() == tfb_int4_scales(w.in, w.out, (int)w.group),
             "the scales of a packed weight are those of quantize_int4");
}

// (out, in) padded to whole strips and units
static Tensor expanded(const Int4& w) {
  Tensor out = at::empty({(w.out + 15) / 16 * 16, (w.in + 63) / 64 * 64}, w.scales.options());
  check(tfb_int4_expand(w.codes.data_ptr(), w.scales.data_ptr(), w.in, w.out, (int)w.group, out.data_ptr(),
                        dtype_code(w.scales.scalar_type()), current_stream(w.scales)));
  return out;
}

Tensor int4_expand(const Int4& w) {
  check_plain("Int4Weight.dequantize", {&w.codes, &w.scales});
  BodyGuard guard;
  check_int4(w);
  const c10::cuda::CUDAGuard device(w.scales.device());
  return expanded(w).narrow(0, 0, w.out).narrow(1, 0, w.in).t();
}

// Up to how many rows the products read the packed weights themselves: each 32 rows read and unpack them again, while beyond it
// they are unpacked once, into two parts.  96 and 97 rows, which take the one way and the other: 1024 x 1024 3.9 and 8.2 us, 1024 x
// 4096 10.0 and 12.5, 2048 x 8192 28.6 and 27.5, 1024 x 50304 56.3 and 77.4, 1536 x 6144 12.5 and 19.6; 32 rows more would add a
// third to the first of each pair.
constexpr int64_t kFewRows = 96;

Tensor int4_linear(const Tensor& x, const Int4& w, const Tensor& bias, bool relu, const Tensor& addend_) {
  check_plain("linear_int4", {&x, &w.codes, &w.scales, &bias, &addend_});
  BodyGuard guard;
  check_int4(w);
  TFB_ASSERT(x.defined() && x.dim() >= 1 && x.size(-1) == w.in, "linear_int4: the input's last dimension is the weight's first");
  TFB_ASSERT(x.scalar_type() == w.scales.scalar_type(), "linear_int4: the input has the type of the weight's scales");
  TFB_ASSERT(!bias.defined() || (bias.dim() == 1 && bias.size(0) == w.out && bias.scalar_type() == x.scalar_type()),
             "linear_int4: the bias has one value of the input's type for each column");
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = w.out;
  TFB_ASSERT(!addend_.defined() || (addend_.sizes() == at::IntArrayRef(shape) && addend_.scalar_type() == x.scalar_type()),
             "linear_int4: the addend has the output's shape and the input's type");
  const c10::cuda::CUDAGuard device(x.device());
  Tensor out = at::empty(shape, x.options());
  if (out.numel() == 0) return out;
  Mat a = as_rows(x);
  if (a.s1 != 1 && a.cols > 1) {
    a.keep = a.keep.reshape({a.rows, a.cols}).contiguous();
    a.p = a.keep.data_ptr();
    a.s0 = a.cols;
  }
  a.s1 = 1;
  const Tensor b = bias.defined() ? bias.contiguous() : Tensor();
  const int dtype = dtype_code(x.scalar_type());
  const cudaStream_t stream = current_stream(x);
  Tensor addend;
  if (addend_.defined()) addend = addend_.contiguous();
  if (a.rows <= kFewRows) {
    check(tfb_int4_linear(a.p, a.rows > 1 ? a.s0 : a.cols, w.codes.data_ptr(), w.scales.data_ptr(), b.defined() ? b.data_ptr() : nullptr,
                          addend.defined() ? addend.data_ptr() : nullptr, w.out, out.data_ptr(), w.out, a.rows, w.in, w.out,
                          (int)w.group, relu ? 1 : 0, dtype, stream));
    return out;
  }
  // More: each weight as the sum of two numbers that it has 16 bits for, along a contraction of twice the length, in one product.
  const int64_t inner = (w.in + 63) / 64 * 64 * 2;
  const Tensor parts = at::empty({(w.out + 15) / 16 * 16, inner}, x.options()), twice = at::empty({a.rows, inner}, x.options());
  check(tfb_int4_split(w.codes.data_ptr(), w.scales.data_ptr(), w.in, w.out, (int)w.group, parts.data_ptr(), a.p, a.s0, a.rows,
                       twice.data_ptr(), dtype, stream));
  Mat k = block(parts.data_ptr(), w.out, inner).t();
  Epilogue e;
  e.bias = b.defined() ? b.data_ptr() : nullptr;
  e.relu = relu;
  e.addend = addend.defined() ? addend.data_ptr() : nullptr;
  e.ld_addend = w.out;
  gemm(block(twice.data_ptr(), a.rows, inner), k, out.data_ptr(), w.out, e, dtype, x.device(), stream);
  return out;
}

static Tensor each_row(const Setting& s, int64_t rows, at::ScalarType type, const char* what) {
  if (!s.each.defined()) return Tensor();
  if (!(s.each.dim() == 1 && s.each.size(0) == rows && s.each.scalar_type() == type))
    throw ArgumentError(std::string("sample_tokens: ") + what + (type == at::kInt ? ": expected a number or a (batch,) int32 tensor"
                                                                                 : ": expected a number or a (batch,) fp32 tensor"));
  return s.each.contiguous();
}
template <typename V>
static const V* values(const Tensor& t) { return t.defined() ? static_cast<const V*>(t.data_ptr()) : nullptr; }

Tensor sample(const Tensor& logits_, const Tensor& uniforms_, const Setting& temperature, const Setting& top_k, const Setting& top_p,
              const Setting& min_p) {
  check_plain("sample_tokens", {&logits_, &uniforms_, &temperature.each, &top_k.each, &top_p.each, &min_p.each});
  BodyGuard guard;
  TFB_ASSERT(logits_.defined() && logits_.dim() == 2 && logits_.size(1) > 0, "sample_tokens: the logits are a (batch, vocab) tensor");
  TFB_ASSERT(is_16_bit(logits_.scalar_type()) || logits_.scalar_type() == at::kFloat, "sample_tokens expects fp16, bf16 or fp32 logits");
  const int64_t B = logits_.size(0), vocab = logits_.size(1);
  TFB_ASSERT(uniforms_.defined() && uniforms_.dim() == 1 && uniforms_.size(0) == B && uniforms_.scalar_type() == at::kFloat,
             "sample_tokens: the uniform numbers are a (batch,) fp32 tensor");
  const Tensor t = each_row(temperature, B, at::kFloat, "temperature"), k = each_row(top_k, B, at::kInt, "top_k"),
               p = each_row(top_p, B, at::kFloat, "top_p"), m = each_row(min_p, B, at::kFloat, "min_p");
  TFB_ASSERT(std::isfinite(temperature.all) && temperature.all >= 0, "sample_tokens: temperature: expected a finite number from 0 on");
  TFB_ASSERT(top_k.all >= 0 && top_k.all < (1LL << 31) && top_k.all == std::floor(top_k.all),
             "sample_tokens: top_k: expected a whole number from 0 (all) on");
  TFB_ASSERT(top_p.all > 0 && top_p.all <= 1, "sample_tokens: top_p: expected a number above 0, up to 1");
  TFB_ASSERT(min_p.all >= 0 && min_p.all <= 1, "sample_tokens: min_p: expected a number from 0 to 1");
  const c10::cuda::CUDAGuard device(logits_.device());
  Tensor out = at::empty({B}, logits_.options().dtype(at::kLong));
  if (B == 0) return out;
  const Tensor logits = vocab > 1 && logits_.stride(1) != 1 ? logits_.contiguous() : logits_, uniforms = uniforms_.contiguous();
  check(tfb_sample(logits.data_ptr(), B > 1 ? logits.stride(0) : vocab, values<float>(uniforms), values<float>(t), (float)temperature.all,
                   values<int>(k), (int)top_k.all, values<float>(p), (float)top_p.all, values<float>(m), (float)min_p.all,
                   static_cast<int64_t*>(out.data_ptr()), B, vocab, dtype_code(logits.scalar_type()), current_stream(logits)));
  return out;
}

}  // namespace tfb_host
