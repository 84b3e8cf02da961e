// The hot torch.library ops (mxf8::quant_rows, adaln_quant_rows, gemm_rowwise, lora_down,
// attn_quant_kv, attn_fwd_q, rotary_table, rotate_qk, gated_residual_norm, mxfp4_quant,
// mxfp4_dequant, gemm_mxfp4, mxfp4_linear, kv_append, kv_read, kv_attend) as native kernels over the C ABI of
// libmxf8.  Their schemas and
// fake kernels are declared in minimaxh3_amd/ops.py; the kernels here take the CUDA and
// AutogradCUDA entries of the dispatcher (the device type of a ROCm GPU), where they stand in
// for the Python kernels of the declarations.
//
// What this path costs is what a short call costs: a Python op body (dispatch through two
// Python kernels, checks, ctypes) took about 20 us per launch, more than most launches of a
// few hundred tokens run on the GPU.  On an MI355X host, one FP8Linear call (two launches)
// 42.5 -> 16.4 us, one short attention call (four launches) 60.6 -> 33.5 us.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/ExpandUtils.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <atomic>

#include "../../include/mxf8.h"

namespace {

using at::Tensor;
using std::optional;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A non-zero status of the C ABI raises minimaxh3_amd._native.NativeError with the library's
// message (of this thread).
void check(int rc, const char* what) {
  if (rc == 0) return;
  const PyGILState_STATE gil = PyGILState_Ensure();
  PyObject* mod = PyImport_ImportModule("minimaxh3_amd._native");
  PyObject* res = mod ? PyObject_CallMethod(mod, "check", "is", rc, what) : nullptr;
  Py_XDECREF(res);
  Py_XDECREF(mod);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (status %d)", what, rc);
  python_error err;
  err.persist();
  PyGILState_Release(gil);
  throw err;
}

// The kernels are built for gfx950 only (checked once per device).
void require_gfx950(const Tensor& t, const char* what) {
  constexpr int kMax = 64;
  static std::atomic<int> known[kMax];
  TORCH_CHECK_VALUE(t.is_cuda(), what, ": expected a GPU tensor");
  const int idx = t.get_device();
  int ok = idx < kMax ? known[idx].load(std::memory_order_relaxed) : 0;
  if (ok == 0) {
    hipDeviceProp_t p;
    const bool gfx950 =
        hipGetDeviceProperties(&p, idx) == hipSuccess && std::string(p.gcnArchName).substr(0, 6) == "gfx950" &&
        (p.gcnArchName[6] == 0 || p.gcnArchName[6] == ':');
    ok = gfx950 ? 1 : 2;
    if (idx < kMax) known[idx].store(ok, std::memory_order_relaxed);
  }
  TORCH_CHECK(ok == 1, "minimaxh3_amd kernels need a gfx950 (MI355X) device, got cuda:", idx);
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return MXF8_BF16;
    case at::kHalf: return MXF8_F16;
    case at::kFloat: return MXF8_F32;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t.scalar_type());
  }
}

void on_device(const Tensor& t, at::Device dev, const char* what, const char* name) {
  TORCH_CHECK_VALUE(t.device() == dev, what, name, " must be on ", dev, ", got ", t.device());
}

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dt) {
  return at::empty(sizes, like.options().dtype(dt));
}

// The same straight from the caching allocator: a kernel that writes all of it and costs a few us should not go through
// the dispatcher for each output.
Tensor fresh(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dt) {
  return at::detail::empty_cuda(sizes, dt, like.device(), std::nullopt);
}

// As at::empty_like: the dimensions in x's memory order.
Tensor fresh_like(const Tensor& x) {
  const std::vector<int64_t> strides =
      x.is_non_overlapping_and_dense() ? x.strides().vec() : at::infer_dense_strides(x.sizes(), x.strides());
  return at::detail::empty_strided_cuda(x.sizes(), strides, x.scalar_type(), x.device());
}

constexpr auto kE4M3 = at::kFloat8_e4m3fn;

std::tuple<Tensor, Tensor> quant_rows(const Tensor& x_in) {
  require_gfx950(x_in, "quant_rows");
  TORCH_CHECK_INDEX(x_in.dim() >= 2, "quant_rows: expected x [M, K], got ", x_in.dim(), " dimensions");
  TORCH_CHECK_VALUE(x_in.dim() == 2, "quant_rows: expected x [M, K]");
  const Tensor x = x_in.stride(1) != 1 || x_in.stride(0) < x_in.size(1) ? x_in.contiguous() : x_in;
  const int64_t M = x.size(0), K = x.size(1);
  Tensor x8 = empty({M, K}, x, kE4M3), scale = empty({M, 1}, x, at::kFloat);
  if (M > 0) {
    const c10::DeviceGuard guard(x.device());
    check(mxf8_quant_rows(x.data_ptr(), dtype_code(x), M, K, std::max(x.stride(0), K),
                          static_cast<uint8_t*>(x8.data_ptr()), scale.data_ptr<float>(), stream_of(x)),
          "quant_rows");
  }
  return {x8, scale};
}

std::tuple<Tensor, Tensor, Tensor> adaln_quant_rows(const Tensor& x, const Tensor& shift_in, const Tensor& scale_in,
                                                    double eps, bool eager, bool want_y) {
  require_gfx950(x, "adaln_quant_rows");
  TORCH_CHECK_VALUE(x.dim() == 3 && shift_in.dim() == 2 && shift_in.size(0) == x.size(0) &&
                        shift_in.size(1) == x.size(2) && scale_in.sizes() == shift_in.sizes(),
                    "adaln_quant_rows: expected x [B, S, C] and shift, scale [B, C]");
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && shift_in.scalar_type() == at::kBFloat16 &&
                        scale_in.scalar_type() == at::kBFloat16,
                    "adaln_quant_rows: bf16 tensors expected");
  on_device(shift_in, x.device(), "adaln_quant_rows: ", "shift");
  on_device(scale_in, x.device(), "adaln_quant_rows: ", "scale");
  const int64_t B = x.size(0), S = x.size(1), C = x.size(2), M = B * S;
  Tensor x2 = x.reshape({M, C}), shift = shift_in, scale = scale_in;
  if (x2.stride(1) != 1) x2 = x2.contiguous();
  // one row stride for both (expanded / strided operands are copied)
  if (shift.stride(1) != 1 || shift.stride(0) < C || shift.stride(0) % 8) shift = shift.contiguous();
  if (scale.stride(1) != 1 || scale.stride(0) != shift.stride(0)) {
    scale = scale.contiguous();
    if (scale.stride(0) != shift.stride(0)) shift = shift.contiguous();
  }
  Tensor x8 = empty({M, C}, x, kE4M3), sa = empty({M, 1}, x, at::kFloat);
  Tensor y = want_y ? empty({M, C}, x, at::kBFloat16) : empty({0}, x, at::kBFloat16);
  if (M > 0) {
    const c10::DeviceGuard guard(x.device());
    check(mxf8_adaln_quant_rows(x2.data_ptr(), M, C, x2.stride(0), S, shift.data_ptr(), scale.data_ptr(),
                                shift.stride(0), static_cast<float>(eps), eager, static_cast<uint8_t*>(x8.data_ptr()),
                                sa.data_ptr<float>(), want_y ? y.data_ptr() : nullptr, stream_of(x)),
          "adaln_quant_rows");
  }
  return {x8, sa, y};
}

Tensor gemm_rowwise(const Tensor& a8, const Tensor& w8, const Tensor& sa, const Tensor& sw,
                    const optional<Tensor>& bias, int64_t act, const optional<Tensor>& lora_t,
                    const optional<Tensor>& lora_b, double lora_scale) {
  const char* what = "gemm_rowwise: ";
  require_gfx950(a8, "gemm_rowwise");
  TORCH_CHECK_VALUE(a8.dim() == 2 && a8.scalar_type() == kE4M3 && w8.scalar_type() == kE4M3 && w8.dim() == 2 &&
                        w8.size(1) == a8.size(1),
                    what, "e4m3 a8 [M, K] and w8 [N, K] expected, got ", a8.scalar_type(), " ", a8.sizes(), " and ",
                    w8.scalar_type(), " ", w8.sizes());
  const int64_t M = a8.size(0), K = a8.size(1), N = w8.size(0);
  TORCH_CHECK_VALUE(a8.is_contiguous() && w8.is_contiguous(), what, "a8 and w8 must be contiguous");
  TORCH_CHECK_VALUE(sa.scalar_type() == at::kFloat && sa.numel() == M && sw.scalar_type() == at::kFloat &&
                        sw.numel() == N,
                    what, "fp32 scales of ", M, " rows and ", N, " channels expected");
  TORCH_CHECK_VALUE(sa.is_contiguous() && sw.is_contiguous(), what, "scales must be contiguous");
  TORCH_CHECK_VALUE(!bias || (bias->scalar_type() == at::kBFloat16 && bias->numel() == N && bias->is_contiguous()),
                    what, "bias must be ", N, " contiguous bf16 values");
  TORCH_CHECK_VALUE(!lora_t || (lora_b && lora_t->dim() == 2 && lora_t->size(0) == M && lora_b->dim() == 2 &&
                                lora_b->size(0) == N && lora_b->size(1) == lora_t->size(1) &&
                                lora_t->scalar_type() == at::kBFloat16 && lora_b->scalar_type() == at::kBFloat16 &&
                                lora_t->is_contiguous() && lora_b->is_contiguous()),
                    what, "LoRA operands t [M, r] and B [N, r] (contiguous bf16) expected");
  const at::Device dev = a8.device();
  on_device(w8, dev, what, "w8");
  on_device(sa, dev, what, "sa");
  on_device(sw, dev, what, "sw");
  if (bias) on_device(*bias, dev, what, "bias");
  if (lora_t) on_device(*lora_t, dev, what, "lora_t");
  if (lora_b) on_device(*lora_b, dev, what, "lora_b");
  Tensor out = empty({M, N}, a8, at::kBFloat16);
  if (M == 0 || N == 0) return out;
  const c10::DeviceGuard guard(dev);
  check(mxf8_gemm_rowwise(static_cast<const uint8_t*>(a8.data_ptr()), static_cast<const uint8_t*>(w8.data_ptr()),
                          sa.data_ptr<float>(), sw.data_ptr<float>(), bias ? bias->data_ptr() : nullptr,
                          static_cast<int>(act), lora_t ? lora_t->data_ptr() : nullptr,
                          lora_b ? lora_b->data_ptr() : nullptr, lora_t ? lora_t->size(1) : 0,
                          static_cast<float>(lora_scale), out.data_ptr(), M, N, K, N, stream_of(a8)),
        "gemm_rowwise");
  return out;
}

Tensor lora_down(const Tensor& x_in, const Tensor& a_in) {
  require_gfx950(x_in, "lora_down");
  TORCH_CHECK_INDEX(x_in.dim() >= 2, "lora_down: expected x [M, K], got ", x_in.dim(), " dimensions");
  // (the kernel reads both as bf16 and addresses A by x's K)
  TORCH_CHECK_VALUE(x_in.dim() == 2 && a_in.dim() == 2 && a_in.size(1) == x_in.size(1) &&
                        x_in.scalar_type() == at::kBFloat16 && a_in.scalar_type() == at::kBFloat16,
                    "lora_down: bf16 x [M, K] and A [r, K] expected, got ", x_in.scalar_type(), " ", x_in.sizes(),
                    " and ", a_in.scalar_type(), " ", a_in.sizes());
  on_device(a_in, x_in.device(), "lora_down: ", "a");
  const Tensor x = x_in.stride(1) != 1 ? x_in.contiguous() : x_in, a = a_in.contiguous();
  const int64_t M = x.size(0), K = x.size(1), r = a.size(0);
  Tensor t = empty({M, r}, x, at::kBFloat16);
  if (M > 0) {
    const c10::DeviceGuard guard(x.device());
    check(mxf8_lora_down(x.data_ptr(), x.stride(0), a.data_ptr(), t.data_ptr(), M, K, r, stream_of(x)), "lora_down");
  }
  return t;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> attn_quant_kv(const Tensor& k, const Tensor& v) {
  require_gfx950(k, "attn_quant_kv");
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() &&
                        k.device() == v.device(),
                    "attn_quant_kv: k and v must have one shape, dtype and device");
  const int64_t B = k.size(0), H = k.size(1), S = k.size(2), D = k.size(3), nk = cdiv(S, 128);
  Tensor k8 = empty({B, H, nk * 128, D}, k, kE4M3), sk = empty({B, H, nk}, k, at::kFloat);
  Tensor v8t = empty({B, H, D, nk * 128}, k, kE4M3), sv = empty({B, H, D}, k, at::kFloat);
  Tensor mean = empty({B, H, D}, k, at::kFloat);
  Tensor ws = empty({std::max<int64_t>(mxf8_attn_kv_workspace_bytes(B, H, S, D), 16)}, k, at::kByte);
  const c10::DeviceGuard guard(k.device());
  check(mxf8_attn_quant_kv(k.data_ptr(), k.strides().data(), v.data_ptr(), v.strides().data(), dtype_code(k), B, H, S,
                           D, static_cast<uint8_t*>(k8.data_ptr()), sk.data_ptr<float>(),
                           static_cast<uint8_t*>(v8t.data_ptr()), sv.data_ptr<float>(), mean.data_ptr<float>(),
                           ws.data_ptr(), stream_of(k)),
        "attn_quant_kv");
  return {k8, sk, v8t, sv, mean};
}

// The K/V codes must have exactly the layout attn_quant_kv gives for Sk keys (the kernels
// address them through Sk alone).
void check_codes(const Tensor& t, at::IntArrayRef shape, at::ScalarType dt, const char* name, int64_t Sk,
                 at::Device dev) {
  TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == dt && t.is_contiguous(), "attn_fwd_q: ", name,
                    " must be a contiguous ", dt, " tensor of shape ", shape, " for Sk=", Sk, ", got ",
                    t.scalar_type(), " ", t.sizes());
  on_device(t, dev, "attn_fwd_q: ", name);
}

// key_mask (bool) / key_bias (fp32) as one row of Sk values per batch item.
Tensor key_operand(const Tensor& t_in, at::ScalarType dt, const char* name, int64_t B, int64_t Sk, at::Device dev) {
  on_device(t_in, dev, "", name);
  Tensor t = t_in.to(dt);
  if (t.numel() == B * Sk)
    t = t.reshape({B, Sk});
  else if (t.numel() == Sk)
    t = t.reshape({1, Sk}).expand({B, Sk});
  else
    TORCH_CHECK_VALUE(false, name, " must hold B*Sk = ", B * Sk, " (or Sk = ", Sk, ") values, got shape ", t.sizes());
  return t.contiguous();
}

// As ops.attn_fwd_q_supported, for a 4-d q.
bool fused_q_layout(const Tensor& q) {
  return (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && q.stride(3) == 1 &&
         q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && q.stride(2) % 8 == 0;
}

Tensor attn_fwd_q(const Tensor& q, double c, const Tensor& k8, const Tensor& v8t, const Tensor& sk, const Tensor& sv,
                  const optional<Tensor>& key_mask, const optional<Tensor>& key_bias, double repair_tau, int64_t Sk,
                  int64_t kv_mode) {
  require_gfx950(q, "attn_fwd_q");
  TORCH_CHECK_VALUE(q.dim() == 4 && fused_q_layout(q),
                    "attn_fwd_q: q must be bf16/fp16 with unit channel stride, other strides multiples of 8 and "
                    "16-byte alignment");
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16) {
    // a view that starts off a 16-byte boundary: the two launches give the same bits
    static const auto quant_q = c10::Dispatcher::singleton()
                                    .findSchemaOrThrow("mxf8::attn_quant_q", "")
                                    .typed<std::tuple<Tensor, Tensor>(const Tensor&, double)>();
    static const auto fwd =
        c10::Dispatcher::singleton()
            .findSchemaOrThrow("mxf8::attn_fwd", "")
            .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                          const optional<Tensor>&, const optional<Tensor>&, double, const Tensor&, int64_t, int64_t)>();
    const auto [q8, sq] = quant_q.call(q, c);
    return fwd.call(q8, k8, v8t, sq, sk, sv, key_mask, key_bias, repair_tau, q, Sk, kv_mode);
  }
  const int64_t B = q.size(0), H = q.size(1), Sq = q.size(2), D = q.size(3), Skp = cdiv(Sk, 128) * 128;
  const at::Device dev = q.device();
  check_codes(k8, {B, H, Skp, D}, kE4M3, "k8", Sk, dev);
  check_codes(v8t, {B, H, D, Skp}, kE4M3, "v8t", Sk, dev);
  check_codes(sk, {B, H, Skp / 128}, at::kFloat, "sk", Sk, dev);
  check_codes(sv, {B, H, D}, at::kFloat, "sv", Sk, dev);
  Tensor out = at::empty_like(q), km, kb;
  if (key_mask) km = key_operand(*key_mask, at::kBool, "key_mask", B, Sk, dev);
  if (key_bias) kb = key_operand(*key_bias, at::kFloat, "key_bias", B, Sk, dev);
  const c10::DeviceGuard guard(dev);
  check(mxf8_attn_fwd_q(q.data_ptr(), q.strides().data(), static_cast<float>(c),
                        static_cast<const uint8_t*>(k8.data_ptr()), static_cast<const uint8_t*>(v8t.data_ptr()),
                        sk.data_ptr<float>(), sv.data_ptr<float>(),
                        km.defined() ? static_cast<const uint8_t*>(km.data_ptr()) : nullptr,
                        kb.defined() ? kb.data_ptr<float>() : nullptr, static_cast<float>(repair_tau), nullptr,
                        out.data_ptr(), dtype_code(out), out.strides().data(), B, H, Sq, Sk, D,
                        static_cast<int>(kv_mode), stream_of(q)),
        "attn_fwd_q");
  return out;
}

// ---- rotary positions, gated residual norms, 4-bit linear -------------------------------------

Tensor rotary_table(const Tensor& positions, at::IntArrayRef axis_dims, double theta) {
  require_gfx950(positions, "rotary_table");
  const int64_t axes = static_cast<int64_t>(axis_dims.size());
  TORCH_CHECK_VALUE(positions.dim() >= 2 && positions.size(-1) == axes, "rotary_table: positions [..., ", axes,
                    "] expected for ", axes, " axes, got ", positions.sizes());
  int type;
  switch (positions.scalar_type()) {
    case at::kFloat: type = 0; break;
    case at::kDouble: type = 1; break;
    case at::kInt: type = 2; break;
    case at::kLong: type = 3; break;
    default: TORCH_CHECK_VALUE(false, "rotary_table: positions must be fp32, fp64, int32 or int64, got ",
                               positions.scalar_type());
  }
  int64_t pairs = 0;
  for (const int64_t d : axis_dims) {
    TORCH_CHECK_VALUE(d > 0 && d % 2 == 0 && d <= 512, "rotary_table: axis dimensions must be even and positive, got ",
                      axis_dims);
    pairs += d / 2;
  }
  const Tensor pos = positions.contiguous();
  std::vector<int64_t> shape(positions.sizes().begin(), positions.sizes().end() - 1);
  shape.push_back(pairs);
  shape.push_back(2);
  Tensor table = fresh(shape, pos, at::kFloat);
  const c10::DeviceGuard guard(pos.device());
  check(mxf8_rotary_table(pos.data_ptr(), type, axes ? pos.numel() / axes : 0, axes, axis_dims.data(), theta,
                          table.data_ptr<float>(), stream_of(pos)),
        "rotary_table");
  return table;
}

// x with contiguous channels (a copy where they are not).
Tensor rows_of(const Tensor& x) { return x.size(-1) > 1 && x.stride(-1) != 1 ? x.contiguous() : x; }

void check_weight(const optional<Tensor>& w, int64_t n, const Tensor& x, const char* what, const char* name) {
  if (!w) return;
  TORCH_CHECK_VALUE(w->dim() == 1 && w->numel() == n && w->scalar_type() == x.scalar_type() && w->is_contiguous(), what,
                    name, " must be ", n, " contiguous ", x.scalar_type(), " values, got ", w->scalar_type(), " ",
                    w->sizes());
  on_device(*w, x.device(), what, name);
}

std::tuple<Tensor, Tensor> rotate_qk(const Tensor& q_in, const optional<Tensor>& k_in, const Tensor& table,
                                     const optional<Tensor>& q_weight, const optional<Tensor>& k_weight, double eps,
                                     bool interleaved) {
  const char* what = "rotate_qk: ";
  require_gfx950(q_in, "rotate_qk");
  TORCH_CHECK_VALUE(q_in.dim() == 4, what, "q must be [B, H, S, D], got ", q_in.sizes());
  const int64_t B = q_in.size(0), Hq = q_in.size(1), S = q_in.size(2), D = q_in.size(3);
  const at::Device dev = q_in.device();
  dtype_code(q_in);
  if (k_in) {
    TORCH_CHECK_VALUE(k_in->dim() == 4 && k_in->size(0) == B && k_in->size(2) == S && k_in->size(3) == D, what,
                      "k must be [B, Hk, S, D] with q's B, S and D, got ", k_in->sizes(), " for q ", q_in.sizes());
    TORCH_CHECK_VALUE(k_in->scalar_type() == q_in.scalar_type(), what, "q and k must have one dtype");
    on_device(*k_in, dev, what, "k");
  }
  TORCH_CHECK_VALUE(k_in || !k_weight, what, "k_weight needs k");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kFloat && table.is_contiguous() &&
                        (table.dim() == 3 || (table.dim() == 4 && table.size(0) == B)) && table.size(-1) == 2 &&
                        table.size(-3) == S && 2 * table.size(-2) <= D,
                    what, "table must be contiguous fp32 [S, P, 2] or [B, S, P, 2] with 2 P <= D, got ",
                    table.scalar_type(), " ", table.sizes(), " for q ", q_in.sizes());
  on_device(table, dev, what, "table");
  check_weight(q_weight, D, q_in, what, "q_weight");
  check_weight(k_weight, D, q_in, what, "k_weight");
  const Tensor q = rows_of(q_in), k = k_in ? rows_of(*k_in) : Tensor();
  Tensor qo = fresh_like(q), ko = k_in ? fresh_like(k) : fresh({0}, q, q.scalar_type());
  if (qo.stride(3) != 1) qo = at::empty(q.sizes(), q.options());
  if (k_in && ko.stride(3) != 1) ko = at::empty(k.sizes(), k.options());
  const int64_t P = table.size(-2);
  const c10::DeviceGuard guard(dev);
  check(mxf8_rotate_qk(q.data_ptr(), q.strides().data(), Hq, k_in ? k.data_ptr() : nullptr,
                       k_in ? k.strides().data() : nullptr, k_in ? k.size(1) : 0, dtype_code(q), B, S, D,
                       table.data_ptr<float>(), table.dim() == 4 ? S * P * 2 : 0, P,
                       q_weight ? q_weight->data_ptr() : nullptr, k_weight ? k_weight->data_ptr() : nullptr,
                       static_cast<float>(eps), interleaved, qo.data_ptr(), qo.strides().data(),
                       k_in ? ko.data_ptr() : nullptr, k_in ? ko.strides().data() : nullptr, stream_of(q)),
        "rotate_qk");
  return {qo, ko};
}

// Modulation rows [B, C] or [B, G, C]: their number per item, and the strides of item and row.
struct ModRows {
  Tensor t;
  int64_t batch = 0, span = 0;
  const void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_residual_norm(
    const Tensor& x_in, const optional<Tensor>& branch_in, const optional<Tensor>& gate, const optional<Tensor>& shift,
    const optional<Tensor>& scale, const optional<Tensor>& branch_weight, const optional<Tensor>& weight, bool layer,
    double eps, double residual_scale, int64_t quant, bool want_y) {
  const char* what = "gated_residual_norm: ";
  require_gfx950(x_in, "gated_residual_norm");
  TORCH_CHECK_VALUE(x_in.dim() == 3, what, "x must be [B, S, C], got ", x_in.sizes());
  const int64_t B = x_in.size(0), S = x_in.size(1), C = x_in.size(2), M = B * S;
  const at::Device dev = x_in.device();
  const int dt = dtype_code(x_in);
  TORCH_CHECK_VALUE(C > 0, what, "x has no channels");
  if (branch_in) {
    TORCH_CHECK_VALUE(branch_in->sizes() == x_in.sizes() && branch_in->scalar_type() == x_in.scalar_type(), what,
                      "branch must have x's shape and dtype, got ", branch_in->scalar_type(), " ", branch_in->sizes());
    on_device(*branch_in, dev, what, "branch");
  }
  TORCH_CHECK_VALUE(branch_in || (!gate && !branch_weight), what, "gate and branch_weight need a branch");
  check_weight(branch_weight, C, x_in, what, "branch_weight");
  check_weight(weight, C, x_in, what, "weight");
  TORCH_CHECK_VALUE(quant >= MXF8_QUANT_NONE && quant <= MXF8_QUANT_MXFP4, what, "bad quantization ", quant);
  TORCH_CHECK_VALUE(quant != MXF8_QUANT_MXFP4 || C % 32 == 0, what, "C = ", C, " must be a multiple of 32 for mxfp4");
  int64_t spans = 0;
  auto rows = [&](const optional<Tensor>& t, const char* name) {
    ModRows m;
    if (!t) return m;
    TORCH_CHECK_VALUE((t->dim() == 2 || t->dim() == 3) && t->size(0) == B && t->size(-1) == C &&
                          t->scalar_type() == x_in.scalar_type(),
                      what, name, " must be [B, C] or [B, G, C] of x's dtype, got ", t->scalar_type(), " ", t->sizes());
    on_device(*t, dev, what, name);
    const int64_t g = t->dim() == 3 ? t->size(1) : 1;
    TORCH_CHECK_VALUE(spans == 0 || spans == g, what, "gate, shift and scale must have the same number of rows");
    TORCH_CHECK_VALUE(g > 0 && S % g == 0, what, name, " has ", g, " rows per item, which do not divide S = ", S);
    spans = g;
    m.t = rows_of(*t);
    m.batch = m.t.stride(0);
    m.span = m.t.dim() == 3 ? m.t.stride(1) : 0;
    return m;
  };
  const ModRows g = rows(gate, "gate"), sh = rows(shift, "shift"), sc = rows(scale, "scale");
  const Tensor x = rows_of(x_in), br = branch_in ? rows_of(*branch_in) : Tensor();
  Tensor r = fresh(branch_in ? at::IntArrayRef{B, S, C} : at::IntArrayRef{0}, x, x.scalar_type());
  const bool y_out = want_y || quant == MXF8_QUANT_NONE;
  Tensor y = fresh(y_out ? at::IntArrayRef{B, S, C} : at::IntArrayRef{0}, x, x.scalar_type());
  Tensor codes, scales;
  if (quant == MXF8_QUANT_E4M3) {
    codes = fresh({M, C}, x, kE4M3);
    scales = fresh({M, 1}, x, at::kFloat);
  } else if (quant == MXF8_QUANT_MXFP4) {
    codes = fresh({M, C / 2}, x, at::kByte);
    scales = fresh({cdiv(C, 256), M, 8}, x, at::kByte);
  } else {
    codes = fresh({0}, x, at::kByte);
    scales = fresh({0}, x, at::kByte);
  }
  const c10::DeviceGuard guard(dev);
  check(mxf8_gated_residual_norm(x.data_ptr(), x.stride(0), x.stride(1), branch_in ? br.data_ptr() : nullptr,
                                 branch_in ? br.stride(0) : 0, branch_in ? br.stride(1) : 0, dt, B, S, C, g.ptr(),
                                 g.batch, g.span, sh.ptr(), sh.batch, sh.span, sc.ptr(), sc.batch, sc.span,
                                 spans ? spans : 1, branch_weight ? branch_weight->data_ptr() : nullptr,
                                 weight ? weight->data_ptr() : nullptr, layer, static_cast<float>(eps),
                                 static_cast<float>(residual_scale), static_cast<int>(quant),
                                 branch_in ? r.data_ptr() : nullptr, y_out ? y.data_ptr() : nullptr,
                                 quant ? static_cast<uint8_t*>(codes.data_ptr()) : nullptr,
                                 quant ? scales.data_ptr() : nullptr, stream_of(x)),
        "gated_residual_norm");
  return {r, y, codes, scales};
}

std::tuple<Tensor, Tensor> mxfp4_quant(const Tensor& x_in) {
  require_gfx950(x_in, "mxfp4_quant");
  TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.size(1) > 0 && x_in.size(1) % 32 == 0,
                    "mxfp4_quant: x [M, K] with K a multiple of 32 expected, got ", x_in.sizes());
  dtype_code(x_in);
  const Tensor x = x_in.stride(1) != 1 || x_in.stride(0) < x_in.size(1) ? x_in.contiguous() : x_in;
  const int64_t M = x.size(0), K = x.size(1);
  Tensor codes = fresh({M, K / 2}, x, at::kByte), scales = fresh({cdiv(K, 256), M, 8}, x, at::kByte);
  const c10::DeviceGuard guard(x.device());
  check(mxf8_mxfp4_quant(x.data_ptr(), dtype_code(x), M, K, std::max(x.stride(0), K),
                         static_cast<uint8_t*>(codes.data_ptr()), static_cast<uint8_t*>(scales.data_ptr()),
                         stream_of(x)),
        "mxfp4_quant");
  return {codes, scales};
}

// Codes [R, K / 2] and scales of an R-row matrix of K columns.
void check_mxfp4(const Tensor& codes, const Tensor& scales, const char* what, const char* name) {
  TORCH_CHECK_VALUE(codes.dim() == 2 && codes.scalar_type() == at::kByte && codes.size(1) > 0 &&
                        codes.size(1) % 16 == 0 && codes.is_contiguous(),
                    what, name, " codes must be contiguous uint8 [rows, K / 2] with K a multiple of 32, got ",
                    codes.scalar_type(), " ", codes.sizes());
  const std::array<int64_t, 3> want = {cdiv(codes.size(1), 128), codes.size(0), 8};
  TORCH_CHECK_VALUE(scales.sizes() == at::IntArrayRef(want) && scales.scalar_type() == at::kByte && scales.is_contiguous(),
                    what, name, " scales must be contiguous uint8 ", at::IntArrayRef(want), ", got ", scales.scalar_type(),
                    " ", scales.sizes());
  on_device(scales, codes.device(), what, name);
}

Tensor mxfp4_dequant(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  require_gfx950(codes, "mxfp4_dequant");
  check_mxfp4(codes, scales, "mxfp4_dequant: ", "x");
  Tensor out = fresh({codes.size(0), 2 * codes.size(1)}, codes, dtype);
  const c10::DeviceGuard guard(codes.device());
  check(mxf8_mxfp4_dequant(static_cast<const uint8_t*>(codes.data_ptr()), static_cast<const uint8_t*>(scales.data_ptr()),
                           out.size(0), out.size(1), out.data_ptr(), dtype_code(out), stream_of(codes)),
        "mxfp4_dequant");
  return out;
}

Tensor gemm_mxfp4(const Tensor& a4, const Tensor& w4, const Tensor& sa, const Tensor& sw, const optional<Tensor>& bias,
                  int64_t act) {
  const char* what = "gemm_mxfp4: ";
  require_gfx950(a4, "gemm_mxfp4");
  check_mxfp4(a4, sa, what, "activation");
  check_mxfp4(w4, sw, what, "weight");
  TORCH_CHECK_VALUE(a4.size(1) == w4.size(1), what, "activations of K = ", 2 * a4.size(1), " and weights of K = ",
                    2 * w4.size(1));
  const at::Device dev = a4.device();
  on_device(w4, dev, what, "w4");
  const int64_t M = a4.size(0), N = w4.size(0), K = 2 * a4.size(1);
  TORCH_CHECK_VALUE(!bias || (bias->scalar_type() == at::kBFloat16 && bias->numel() == N && bias->is_contiguous()), what,
                    "bias must be ", N, " contiguous bf16 values");
  if (bias) on_device(*bias, dev, what, "bias");
  Tensor out = fresh({M, N}, a4, at::kBFloat16);
  const c10::DeviceGuard guard(dev);
  check(mxf8_gemm_mxfp4(static_cast<const uint8_t*>(a4.data_ptr()), static_cast<const uint8_t*>(w4.data_ptr()),
                        static_cast<const uint8_t*>(sa.data_ptr()), static_cast<const uint8_t*>(sw.data_ptr()),
                        bias ? bias->data_ptr() : nullptr, static_cast<int>(act), out.data_ptr(), M, N, K, N,
                        stream_of(a4)),
        "gemm_mxfp4");
  return out;
}

Tensor mxfp4_linear(const Tensor& x_in, const Tensor& w4, const Tensor& sw, const optional<Tensor>& bias, int64_t act) {
  const char* what = "mxfp4_linear: ";
  require_gfx950(x_in, "mxfp4_linear");
  check_mxfp4(w4, sw, what, "weight");
  const int64_t K = 2 * w4.size(1), N = w4.size(0);
  TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.size(1) == K, what, "x [M, ", K, "] expected, got ", x_in.sizes());
  const at::Device dev = x_in.device();
  on_device(w4, dev, what, "w4");
  TORCH_CHECK_VALUE(!bias || (bias->scalar_type() == at::kBFloat16 && bias->numel() == N && bias->is_contiguous()), what,
                    "bias must be ", N, " contiguous bf16 values");
  if (bias) on_device(*bias, dev, what, "bias");
  const Tensor x = x_in.stride(1) != 1 || x_in.stride(0) < K ? x_in.contiguous() : x_in;
  const int dt = dtype_code(x);
  const int64_t M = x.size(0), ws = mxf8_mxfp4_linear_workspace_bytes(M, N, K, dt);
  Tensor out = fresh({M, N}, x, at::kBFloat16), work = ws ? fresh({ws}, x, at::kByte) : Tensor();
  const c10::DeviceGuard guard(dev);
  check(mxf8_mxfp4_linear(x.data_ptr(), dt, std::max(x.stride(0), K), static_cast<const uint8_t*>(w4.data_ptr()),
                          static_cast<const uint8_t*>(sw.data_ptr()), bias ? bias->data_ptr() : nullptr,
                          static_cast<int>(act), out.data_ptr(), M, N, K, N, ws ? work.data_ptr() : nullptr, stream_of(x)),
        "mxfp4_linear");
  return out;
}

// ---- paged e4m3 cache of keys and values ---------------------------------------------------------

// The four tensors of a cache, and a call's page table.
struct Pool {
  int64_t pages, H, page, D;
  Tensor table;
};

Pool pool_of(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& table, int64_t B,
             at::Device dev, const char* what) {
  TORCH_CHECK_VALUE(kc.dim() == 4 && kc.is_contiguous() && vc.is_contiguous() && vc.sizes() == kc.sizes() &&
                        kc.scalar_type() == kE4M3 && vc.scalar_type() == kE4M3,
                    what, "codes must be two contiguous e4m3 tensors [pages, heads, page_size, head_dim], got ",
                    kc.scalar_type(), " ", kc.sizes(), " and ", vc.scalar_type(), " ", vc.sizes());
  TORCH_CHECK_VALUE(ks.sizes() == kc.sizes().slice(0, 2) && vs.sizes() == ks.sizes() && ks.is_contiguous() &&
                        vs.is_contiguous() && ks.scalar_type() == at::kByte && vs.scalar_type() == at::kByte,
                    what, "scales must be two contiguous uint8 tensors [pages, heads], got ", ks.scalar_type(), " ",
                    ks.sizes(), " and ", vs.scalar_type(), " ", vs.sizes());
  TORCH_CHECK_VALUE(table.dim() == 2 && (B < 0 || table.size(0) == B) && table.scalar_type() == at::kInt, what,
                    "page_table must be int32 [B, pages of a sequence], got ", table.scalar_type(), " ", table.sizes());
  for (const Tensor* t : {&kc, &vc, &ks, &vs, &table}) on_device(*t, dev, what, "the cache and its page table");
  const bool rows = (table.stride(1) == 1 || table.size(1) <= 1) && (table.size(0) <= 1 || table.stride(0) >= table.size(1));
  return {kc.size(0), kc.size(1), kc.size(2), kc.size(3), rows ? table : table.contiguous()};
}

void check_per_item(const optional<Tensor>& t, int64_t B, at::Device dev, const char* what, const char* name) {
  if (!t) return;
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == B && t->scalar_type() == at::kInt && t->is_contiguous(), what, name,
                    " must be ", B, " contiguous int32 values, got ", t->scalar_type(), " ", t->sizes());
  on_device(*t, dev, what, name);
}

const int32_t* ints(const optional<Tensor>& t) { return t ? t->data_ptr<int32_t>() : nullptr; }
uint8_t* bytes(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

void kv_append(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& page_table,
               const Tensor& starts, const Tensor& k_in, const Tensor& v_in, const optional<Tensor>& counts,
               const optional<Tensor>& table, const optional<Tensor>& k_weight, double eps, bool interleaved) {
  const char* what = "kv_append: ";
  require_gfx950(k_in, "kv_append");
  TORCH_CHECK_VALUE(k_in.dim() == 4 && v_in.sizes() == k_in.sizes() && v_in.scalar_type() == k_in.scalar_type(), what,
                    "k and v must be [B, H, S, D] of one shape and dtype, got ", k_in.sizes(), " and ", v_in.sizes());
  dtype_code(k_in);
  const at::Device dev = k_in.device();
  on_device(v_in, dev, what, "v");
  const int64_t B = k_in.size(0), H = k_in.size(1), S = k_in.size(2), D = k_in.size(3);
  const Pool p = pool_of(kc, vc, ks, vs, page_table, B, dev, what);
  TORCH_CHECK_VALUE(p.H == H && p.D == D, what, "the cache holds ", p.H, " heads of ", p.D, ", got ", k_in.sizes());
  check_per_item(starts, B, dev, what, "starts");
  check_per_item(counts, B, dev, what, "counts");
  if (table) {
    TORCH_CHECK_VALUE(table->scalar_type() == at::kFloat && table->is_contiguous() &&
                          (table->dim() == 3 || (table->dim() == 4 && table->size(0) == B)) && table->size(-1) == 2 &&
                          table->size(-3) == S && 2 * table->size(-2) <= D,
                      what, "table must be contiguous fp32 [S, P, 2] or [B, S, P, 2] with 2 P <= D, got ",
                      table->scalar_type(), " ", table->sizes(), " for k ", k_in.sizes());
    on_device(*table, dev, what, "table");
  }
  check_weight(k_weight, D, k_in, what, "k_weight");
  const Tensor k = rows_of(k_in), v = rows_of(v_in);
  const int64_t P = table ? table->size(-2) : 0;
  const c10::DeviceGuard guard(dev);
  check(mxf8_kv_append(k.data_ptr(), k.strides().data(), v.data_ptr(), v.strides().data(), dtype_code(k), B, H, S, D,
                       table ? table->data_ptr<float>() : nullptr, table && table->dim() == 4 ? S * P * 2 : 0, P,
                       k_weight ? k_weight->data_ptr() : nullptr, static_cast<float>(eps), interleaved,
                       p.table.data_ptr<int32_t>(), p.table.stride(0), p.table.size(1), starts.data_ptr<int32_t>(),
                       ints(counts), bytes(kc), bytes(vc), bytes(ks), bytes(vs), p.pages, p.page, stream_of(k)),
        "kv_append");
}

std::tuple<Tensor, Tensor> kv_read(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs,
                                   const Tensor& page_table, const Tensor& starts, int64_t tokens,
                                   const optional<Tensor>& lengths, at::ScalarType dtype) {
  const char* what = "kv_read: ";
  require_gfx950(kc, "kv_read");
  const at::Device dev = kc.device();
  const Pool p = pool_of(kc, vc, ks, vs, page_table, -1, dev, what);
  const int64_t B = page_table.size(0);
  check_per_item(starts, B, dev, what, "starts");
  check_per_item(lengths, B, dev, what, "lengths");
  TORCH_CHECK_VALUE(tokens >= 0 && tokens <= (1 << 30), what, "tokens must be from 0 to 2^30, got ", tokens);
  TORCH_CHECK_VALUE(dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat, what, "unsupported dtype ",
                    dtype);
  Tensor k = fresh({B, p.H, tokens, p.D}, kc, dtype), v = fresh({B, p.H, tokens, p.D}, kc, dtype);
  const c10::DeviceGuard guard(dev);
  check(mxf8_kv_read(bytes(kc), bytes(vc), bytes(ks), bytes(vs), p.pages, p.H, p.page, p.D, p.table.data_ptr<int32_t>(),
                     p.table.stride(0), p.table.size(1), B, starts.data_ptr<int32_t>(), tokens, ints(lengths),
                     k.data_ptr(), v.data_ptr(), dtype_code(k), stream_of(kc)),
        "kv_read");
  return {k, v};
}

Tensor kv_attend(const Tensor& q_in, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs,
                 const Tensor& page_table, const Tensor& lengths, const optional<Tensor>& q_lengths, bool causal,
                 double scale) {
  const char* what = "kv_attend: ";
  require_gfx950(q_in, "kv_attend");
  TORCH_CHECK_VALUE(q_in.dim() == 4 && (q_in.scalar_type() == at::kBFloat16 || q_in.scalar_type() == at::kHalf), what,
                    "q must be bf16 or fp16 [B, H, S, D], got ", q_in.scalar_type(), " ", q_in.sizes());
  const at::Device dev = q_in.device();
  const int64_t B = q_in.size(0), H = q_in.size(1), S = q_in.size(2), D = q_in.size(3);
  const Pool p = pool_of(kc, vc, ks, vs, page_table, B, dev, what);
  TORCH_CHECK_VALUE(p.D == D && p.H > 0 && H % p.H == 0, what, "the cache holds ", p.H, " heads of ", p.D, ", got q ",
                    q_in.sizes());
  check_per_item(lengths, B, dev, what, "lengths");
  check_per_item(q_lengths, B, dev, what, "q_lengths");
  const Tensor q = rows_of(q_in);
  Tensor out = fresh_like(q);
  if (out.stride(3) != 1) out = at::empty(q.sizes(), q.options());
  const c10::DeviceGuard guard(dev);
  const int64_t need = mxf8_kv_attend_workspace_bytes(B, H, p.H, S, D, p.table.size(1), p.page);
  Tensor work;
  if (need) work = fresh({need}, q, at::kByte);
  check(mxf8_kv_attend(q.data_ptr(), q.strides().data(), dtype_code(q), B, H, S, D, bytes(kc), bytes(vc), bytes(ks),
                       bytes(vs), p.pages, p.H, p.page, p.table.data_ptr<int32_t>(), p.table.stride(0), p.table.size(1),
                       lengths.data_ptr<int32_t>(), ints(q_lengths), causal, static_cast<float>(scale), out.data_ptr(),
                       out.strides().data(), need ? work.data_ptr() : nullptr, stream_of(q)),
        "kv_attend");
  return out;
}

// The ops have no derivative.  With grad mode on, an output of an input that requires grad
// requires grad and its backward raises; otherwise the call goes on below autograd (as the
// Python declarations' autograd kernel does; forward-mode tangents end here).
void no_derivative(const c10::OperatorHandle& op, c10::DispatchKeySet ks, torch::jit::Stack* stack) {
  const size_t nargs = op.schema().arguments().size();
  torch::autograd::edge_list edges;
  if (at::GradMode::is_enabled()) {
    bool any = false;
    for (size_t i = 0; i < nargs; ++i) {
      const c10::IValue& v = torch::jit::peek(*stack, i, nargs);
      any = any || (v.isTensor() && v.toTensor().defined() && v.toTensor().requires_grad());
    }
    if (any) {
      for (size_t i = 0; i < nargs; ++i) {
        const c10::IValue& v = torch::jit::peek(*stack, i, nargs);
        if (v.isTensor() && v.toTensor().defined() && v.toTensor().requires_grad())
          edges.push_back(torch::autograd::impl::gradient_edge(v.toTensor()));
      }
    }
  }
  {
    const at::AutoDispatchBelowAutograd guard;
    op.redispatchBoxed(ks & c10::after_autograd_keyset, stack);
  }
  if (edges.empty()) return;
  const std::string name = op.schema().name().substr(6);  // without "mxf8::"
  const auto node = std::make_shared<torch::autograd::Error>(
      "Trying to backward through mxf8." + name + ".default but no autograd formula was registered. Please use "
      "register_autograd to add one.", std::move(edges));
  const size_t nret = op.schema().returns().size();
  for (size_t i = 0; i < nret; ++i) {
    const at::Tensor& out = torch::jit::peek(*stack, i, nret).toTensor();
    if (torch::autograd::isDifferentiableType(out.scalar_type())) torch::autograd::set_history(out, node);  // not 4-bit codes
  }
}

}  // namespace

TORCH_LIBRARY_IMPL(mxf8, CUDA, m) {
  m.impl("quant_rows", &quant_rows);
  m.impl("adaln_quant_rows", &adaln_quant_rows);
  m.impl("gemm_rowwise", &gemm_rowwise);
  m.impl("lora_down", &lora_down);
  m.impl("attn_quant_kv", &attn_quant_kv);
  m.impl("attn_fwd_q", &attn_fwd_q);
  m.impl("rotary_table", &rotary_table);
  m.impl("rotate_qk", &rotate_qk);
  m.impl("gated_residual_norm", &gated_residual_norm);
  m.impl("mxfp4_quant", &mxfp4_quant);
  m.impl("mxfp4_dequant", &mxfp4_dequant);
  m.impl("gemm_mxfp4", &gemm_mxfp4);
  m.impl("mxfp4_linear", &mxfp4_linear);
  m.impl("kv_append", &kv_append);
  m.impl("kv_read", &kv_read);
  m.impl("kv_attend", &kv_attend);
}

TORCH_LIBRARY_IMPL(mxf8, AutogradCUDA, m) {
  for (const char* op : {"quant_rows", "adaln_quant_rows", "gemm_rowwise", "lora_down", "attn_quant_kv", "attn_fwd_q",
                         "rotary_table", "rotate_qk", "gated_residual_norm", "mxfp4_quant", "mxfp4_dequant", "gemm_mxfp4",
                         "mxfp4_linear", "kv_append", "kv_read", "kv_attend"})
    m.impl(op, torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
}
