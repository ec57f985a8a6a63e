// Compiled tensor-level binding: the counterpart of the reference's pybind11 module
// torch_dwconv._C (torch_dwconv/dwconv.cpp:60-67) for this library.
//
// It owns nothing but the glue a tensor framework needs around the C ABI of
// include/dwconv_b200.h: argument checks with the reference's texts (CHECK_CUDA,
// dwconv.cpp:24-25), result allocation with the caching allocator, the tensor's device made
// current, the current stream of that device.  All arithmetic is in libdwconv_b200.so, which
// this module links to; no kernel lives here.  dwconv_b200/_C.py holds the same functions
// over ctypes and is what runs when this module has not been built; a call costs a few
// microseconds of host time here and 15-20 there.
//
// Four functions have the reference's names and argument order; `forward` and `backward`
// are what the autograd function calls (one call per direction, both gradients from the
// fused kernel).
#include <torch/extension.h>

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "dwconv_b200.h"

namespace {

std::string shape_text(const at::Tensor &t) {
  // Python's tuple(t.shape) form, so that messages equal the ctypes mirror's
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) {
    s += std::to_string(t.size(i));
    if (i + 1 < t.dim() || t.dim() == 1) s += (i + 1 < t.dim()) ? ", " : ",";
  }
  return s + ")";
}

void check_cuda(const at::Tensor &t, const char *name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
}

int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return DWCONV_B200_F32;
    case at::kHalf: return DWCONV_B200_F16;
    case at::kDouble: return DWCONV_B200_F64;
    case at::kBFloat16: return DWCONV_B200_BF16;
    default:
      TORCH_CHECK(false, "dwconv_b200: unsupported dtype ", t.dtype(),
                  " (float32, float16, bfloat16, float64)");
  }
  return -1;
}

void check_same(const at::Tensor &t, const at::Tensor &o) {
  TORCH_CHECK(o.scalar_type() == t.scalar_type() && o.device() == t.device(),
              "dwconv_b200: tensors must share dtype and device (", t.dtype(), "/", t.device(),
              " vs ", o.dtype(), "/", o.device(), ")");
}

// The library reads C*kh*kw filter values and N*C planes through raw pointers: a tensor of
// another shape would be read out of bounds, so it is refused here.
void check_filter(const at::Tensor &input, const at::Tensor &kernel) {
  TORCH_CHECK(input.dim() == 4 && kernel.dim() == 4, "dwconv_b200: expected 4-d input and kernel, got ",
              shape_text(input), " and ", shape_text(kernel));
  TORCH_CHECK(kernel.size(0) == input.size(1) && kernel.size(1) == 1,
              "dwconv_b200: kernel must be [C, 1, kh, kw] with C = ", input.size(1), ", got ",
              shape_text(kernel));
}

void check_status(int st, const char *what) {
  if (st == DWCONV_B200_OK) return;
  std::string detail = dwconv_b200_status_string(st);
  if (st == 5) detail += " [cudaError " + std::to_string(dwconv_b200_last_cuda_error()) + "]";
  TORCH_CHECK(false, "dwconv_b200.", what, ": ", detail);
}

void *stream_of(const at::Tensor &t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

bool channels_last(const at::Tensor &t) {
  return t.dim() == 4 && !t.is_contiguous() && t.is_contiguous(at::MemoryFormat::ChannelsLast);
}

// what the channels-last kernels cover (other geometries are made contiguous NCHW)
bool nhwc_served(int code, int kh, int kw, int sh, int sw) {
  return kh == kw && (kh == 3 || kh == 5 || kh == 7) && sh == sw && (sh == 1 || sh == 2) &&
         (code == DWCONV_B200_F32 || code == DWCONV_B200_F16 || code == DWCONV_B200_BF16);
}

dwconv_b200_shape make_shape(const at::Tensor &input, const at::Tensor &kernel, int sh, int sw,
                             int ph, int pw, int Ho, int Wo) {
  dwconv_b200_shape s;
  s.N = (int)input.size(0); s.C = (int)input.size(1); s.H = (int)input.size(2); s.W = (int)input.size(3);
  s.kh = (int)kernel.size(2); s.kw = (int)kernel.size(3);
  s.sh = sh; s.sw = sw; s.ph = ph; s.pw = pw; s.Ho = Ho; s.Wo = Wo;
  return s;
}

// ---- what the autograd function calls ------------------------------------------------

// (out, input as read, kernel as read, channels-last?)  The tensors "as read" are what the
// backward must be given: contiguous copies when the arguments were not.
std::tuple<at::Tensor, at::Tensor, at::Tensor, bool> forward(at::Tensor input, at::Tensor kernel,
                                                             int64_t sh, int64_t sw, int64_t ph,
                                                             int64_t pw) {
  check_cuda(input, "input");
  check_cuda(kernel, "kernel");
  const int code = dtype_code(input);
  check_same(input, kernel);
  check_filter(input, kernel);
  const int kh = (int)kernel.size(2), kw = (int)kernel.size(3);
  const bool nhwc = channels_last(input) && nhwc_served(code, kh, kw, (int)sh, (int)sw);
  if (!nhwc) input = input.contiguous();
  kernel = kernel.contiguous();
  const int H = (int)input.size(2), W = (int)input.size(3);
  const int Ho = dwconv_b200_out_size(H, 1, (int)ph, (int)ph, kh, (int)sh);
  const int Wo = dwconv_b200_out_size(W, 1, (int)pw, (int)pw, kw, (int)sw);
  TORCH_CHECK(Ho > 0 && Wo > 0, "depthwise_conv2d: filter ", kh, "x", kw,
              " does not fit the padded input ", H + 2 * ph, "x", W + 2 * pw);
  const dwconv_b200_shape s = make_shape(input, kernel, (int)sh, (int)sw, (int)ph, (int)pw, Ho, Wo);
  at::Tensor out = at::empty({s.N, s.C, Ho, Wo}, input.options(),
                             nhwc ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous);
  c10::cuda::CUDAGuard guard(input.device());
  int st;
  if (nhwc)
    st = dwconv_b200_forward_nhwc(input.data_ptr(), kernel.data_ptr(), out.data_ptr(), code, &s,
                                  nullptr, stream_of(input));
  else
    st = dwconv_b200_forward(input.data_ptr(), kernel.data_ptr(), out.data_ptr(), code, &s,
                             stream_of(input));
  check_status(st, "forward");
  return {out, input, kernel, nhwc};
}

// (grad_input or None, grad_kernel or None) for a forward made by `forward` above.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>> backward(
    const at::Tensor &input, at::Tensor grad_output, const at::Tensor &kernel, int64_t sh, int64_t sw,
    int64_t ph, int64_t pw, bool nhwc, bool want_dx, bool want_dw) {
  const int code = dtype_code(input);
  check_cuda(grad_output, "grad_output");
  check_same(input, grad_output);
  const int kh = (int)kernel.size(2), kw = (int)kernel.size(3);
  const int Ho = dwconv_b200_out_size((int)input.size(2), 1, (int)ph, (int)ph, kh, (int)sh);
  const int Wo = dwconv_b200_out_size((int)input.size(3), 1, (int)pw, (int)pw, kw, (int)sw);
  TORCH_CHECK(grad_output.dim() == 4 && grad_output.size(0) == input.size(0) &&
                  grad_output.size(1) == input.size(1) && grad_output.size(2) == Ho &&
                  grad_output.size(3) == Wo,
              "depthwise_conv2d backward: grad_output has shape ", shape_text(grad_output),
              ", expected (", input.size(0), ", ", input.size(1), ", ", Ho, ", ", Wo, ")");
  const dwconv_b200_shape s = make_shape(input, kernel, (int)sh, (int)sw, (int)ph, (int)pw, Ho, Wo);
  grad_output = grad_output.contiguous(nhwc ? at::MemoryFormat::ChannelsLast
                                            : at::MemoryFormat::Contiguous);
  c10::optional<at::Tensor> dx, dw;
  at::Tensor ws;
  size_t nbytes = 0;
  if (want_dw) {
    nbytes = dwconv_b200_backward_filter_workspace_bytes(code, &s);
    TORCH_CHECK(nbytes != 0, "dwconv_b200.backward: invalid geometry");
    ws = at::empty({(int64_t)nbytes}, input.options().dtype(at::kByte));
    dw = at::empty_like(kernel);
  }
  if (want_dx)
    dx = at::empty_like(input, nhwc ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous);
  c10::cuda::CUDAGuard guard(input.device());
  void *stream = stream_of(input);
  if (nhwc && want_dx && want_dw) {
    check_status(dwconv_b200_backward_nhwc(input.data_ptr(), grad_output.data_ptr(), kernel.data_ptr(),
                                           dx->data_ptr(), dw->data_ptr(), ws.data_ptr(), nbytes, code, &s,
                                           stream),
                 "backward_nhwc");
  } else if (nhwc) {
    if (want_dx)
      check_status(dwconv_b200_backward_input_nhwc(grad_output.data_ptr(), kernel.data_ptr(),
                                                   dx->data_ptr(), code, &s, stream),
                   "backward_input_nhwc");
    if (want_dw)
      check_status(dwconv_b200_backward_filter_nhwc(input.data_ptr(), grad_output.data_ptr(),
                                                    dw->data_ptr(), ws.data_ptr(), nbytes, code, &s,
                                                    stream),
                   "backward_filter_nhwc");
  } else if (want_dx && want_dw) {
    // both gradients from one pass over grad_output
    check_status(dwconv_b200_backward(input.data_ptr(), grad_output.data_ptr(), kernel.data_ptr(),
                                      dx->data_ptr(), dw->data_ptr(), ws.data_ptr(), nbytes, code, &s,
                                      stream),
                 "backward");
  } else if (want_dx) {
    check_status(dwconv_b200_backward_input(grad_output.data_ptr(), kernel.data_ptr(), dx->data_ptr(),
                                            code, &s, stream),
                 "backward_input");
  } else if (want_dw) {
    check_status(dwconv_b200_backward_filter(input.data_ptr(), grad_output.data_ptr(), dw->data_ptr(),
                                             ws.data_ptr(), nbytes, code, &s, stream),
                 "backward_filter");
  }
  return {dx, dw};
}

// ---- the reference's four functions (torch_dwconv/dwconv.cpp:27-67) -------------------

bool use_dwconv2d_small(const at::Tensor &input, const at::Tensor &kernel, int64_t up_h, int64_t up_w,
                        int64_t down_h, int64_t down_w, int64_t pad_h, int64_t pad_w) {
  TORCH_CHECK(input.dim() == 4 && kernel.dim() == 4, "dwconv_b200: expected 4-d input and kernel, got ",
              shape_text(input), " and ", shape_text(kernel));
  return dwconv_b200_use_dwconv2d_small((int)input.size(2), (int)input.size(3), (int)kernel.size(2),
                                        (int)kernel.size(3), (int)up_h, (int)up_w, (int)down_h,
                                        (int)down_w, (int)pad_h, (int)pad_w) != 0;
}

at::Tensor dwconv2d(at::Tensor input, at::Tensor kernel, int64_t up_h, int64_t up_w, int64_t down_h,
                    int64_t down_w, int64_t pad_h0, int64_t pad_h1, int64_t pad_w0, int64_t pad_w1,
                    bool forward_op) {
  check_cuda(input, "input");
  check_cuda(kernel, "kernel");
  const int code = dtype_code(input);
  check_same(input, kernel);
  check_filter(input, kernel);
  input = input.contiguous();
  kernel = kernel.contiguous();
  const int N = (int)input.size(0), C = (int)input.size(1), H = (int)input.size(2), W = (int)input.size(3);
  const int kh = (int)kernel.size(2), kw = (int)kernel.size(3);
  const int oh = dwconv_b200_out_size(H, (int)up_h, (int)pad_h0, (int)pad_h1, kh, (int)down_h);
  const int ow = dwconv_b200_out_size(W, (int)up_w, (int)pad_w0, (int)pad_w1, kw, (int)down_w);
  TORCH_CHECK(oh > 0 && ow > 0, "dwconv_b200.dwconv2d: empty output (", oh, " x ", ow, ")");
  at::Tensor out = at::empty({N, C, oh, ow}, input.options());
  c10::cuda::CUDAGuard guard(input.device());
  check_status(dwconv_b200_dwconv2d(input.data_ptr(), kernel.data_ptr(), out.data_ptr(), code, N, C, H,
                                    W, kh, kw, (int)up_h, (int)up_w, (int)down_h, (int)down_w,
                                    (int)pad_h0, (int)pad_h1, (int)pad_w0, (int)pad_w1,
                                    forward_op ? 1 : 0, stream_of(input)),
               "dwconv2d");
  return out;
}

at::Tensor dwconv2d_small(const at::Tensor &input, const at::Tensor &kernel, int64_t up_h, int64_t up_w,
                          int64_t down_h, int64_t down_w, int64_t pad_h, int64_t pad_w,
                          bool forward_op) {
  return dwconv2d(input, kernel, up_h, up_w, down_h, down_w, pad_h, pad_h, pad_w, pad_w, forward_op);
}

at::Tensor dwconv2d_backward_kernel(at::Tensor input, at::Tensor out_grad, const at::Tensor &kernel,
                                    int64_t up_h, int64_t up_w, int64_t down_h, int64_t down_w,
                                    int64_t pad_h, int64_t pad_w) {
  check_cuda(input, "input");
  check_cuda(out_grad, "out_grad");
  const int code = dtype_code(input);
  check_same(input, out_grad);
  TORCH_CHECK(input.dim() == 4 && out_grad.dim() == 4 && kernel.dim() == 4,
              "dwconv_b200.dwconv2d_backward_kernel: expected 4-d tensors");
  TORCH_CHECK(out_grad.size(0) == input.size(0) && out_grad.size(1) == input.size(1),
              "dwconv_b200.dwconv2d_backward_kernel: out_grad is ", shape_text(out_grad),
              " but input is ", shape_text(input), " (batch and channels must agree)");
  input = input.contiguous();
  out_grad = out_grad.contiguous();
  const int N = (int)input.size(0), C = (int)input.size(1), H = (int)input.size(2), W = (int)input.size(3);
  const int kh = (int)kernel.size(2), kw = (int)kernel.size(3);
  const int oh = (int)out_grad.size(2), ow = (int)out_grad.size(3);
  dwconv_b200_shape s;
  s.N = N; s.C = C; s.H = H; s.W = W; s.kh = kh; s.kw = kw; s.sh = (int)down_h; s.sw = (int)down_w;
  s.ph = (int)pad_h; s.pw = (int)pad_w; s.Ho = oh; s.Wo = ow;
  const size_t nbytes = dwconv_b200_backward_filter_workspace_bytes(code, &s);
  TORCH_CHECK(nbytes != 0, "dwconv_b200.dwconv2d_backward_kernel: invalid geometry");
  at::Tensor dkernel = at::empty({C, 1, kh, kw}, input.options());
  at::Tensor ws = at::empty({(int64_t)nbytes}, input.options().dtype(at::kByte));
  c10::cuda::CUDAGuard guard(input.device());
  check_status(dwconv_b200_dwconv2d_backward_kernel(
                   input.data_ptr(), out_grad.data_ptr(), dkernel.data_ptr(), ws.data_ptr(), nbytes,
                   code, N, C, H, W, oh, ow, kh, kw, (int)up_h, (int)up_w, (int)down_h, (int)down_w,
                   (int)pad_h, (int)pad_w, stream_of(input)),
               "dwconv2d_backward_kernel");
  return dkernel;
}

// ---- sequence operators ----------------------------------------------------------------
// (no counterpart in the reference; the checks' texts equal those of dwconv_b200/sequence.py, which
// has the same functions over ctypes)

using OptTensor = c10::optional<at::Tensor>;

const void *ptr(const OptTensor &t) { return t.has_value() ? t->data_ptr() : nullptr; }

int sequence_dtype(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return DWCONV_B200_F32;
    case at::kHalf: return DWCONV_B200_F16;
    case at::kBFloat16: return DWCONV_B200_BF16;
    default:
      TORCH_CHECK(false, "dwconv_b200: unsupported dtype ", t.dtype(), " (float32, float16, bfloat16)");
  }
  return -1;
}

// channels side by side; any other strides are read as they are
at::Tensor rows_of(const at::Tensor &t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

dwconv_b200_rows rows_arg(const at::Tensor &t) { return {t.data_ptr(), t.stride(0), t.stride(1)}; }

// shape and device of one operand against the input's
void check_operand(const char *fn, const char *name, const at::Tensor &t, at::IntArrayRef shape, at::ScalarType type,
                   const at::Tensor &input) {
  TORCH_CHECK(t.device() == input.device() && t.scalar_type() == type, "dwconv_b200.", fn, ": ", name, " must be ",
              c10::scalarTypeToTypeMeta(type), " on ", input.device(), ", got ", t.dtype(), " on ", t.device());
  if (t.sizes() != shape) {
    std::string want = "(";
    for (size_t i = 0; i < shape.size(); ++i)
      want += std::to_string(shape[i]) + (i + 1 < shape.size() ? ", " : shape.size() == 1 ? "," : "");
    TORCH_CHECK(false, "dwconv_b200.", fn, ": ", name, " must be ", want, "), got ", shape_text(t));
  }
}

// What the forward call left for this one, and hooks on saved tensors may have had in hand since.
void check_kept(const char *fn, const char *name, const at::Tensor &t, at::IntArrayRef shape, const at::Tensor &input) {
  check_operand(fn, name, t, shape, at::kFloat, input);
  TORCH_CHECK(t.is_contiguous(), "dwconv_b200.", fn, ": ", name, " must be contiguous");
}

dwconv_b200_sequence check_sequences(const char *fn, const at::Tensor &input, const OptTensor &offsets) {
  check_cuda(input, "input");
  sequence_dtype(input);
  TORCH_CHECK(input.dim() == 3, "dwconv_b200.", fn, ": expected input [B, T, C], got ", shape_text(input));
  for (int d = 0; d < 3; ++d)
    TORCH_CHECK(input.size(d) <= (1ll << 30), "dwconv_b200.", fn, ": input is too large: ", shape_text(input));
  dwconv_b200_sequence s{(int)input.size(0), (int)input.size(1), (int)input.size(2), nullptr, 0};
  if (offsets.has_value()) {
    const at::Tensor &o = *offsets;
    TORCH_CHECK(o.device() == input.device() && o.scalar_type() == at::kInt && o.dim() == 1 && o.is_contiguous() &&
                    o.size(0) >= 2,
                "dwconv_b200.", fn, ": offsets must be a contiguous 1-d int32 tensor of at least 2 row numbers on ",
                input.device());
    TORCH_CHECK(s.B == 1, "dwconv_b200.", fn, ": packed sequences (offsets) need a batch of 1, got ", s.B);
    s.offsets = o.data_ptr();
    s.S = (int)o.size(0) - 1;
  }
  return s;
}

int64_t state_count(const dwconv_b200_sequence &s) { return s.offsets ? s.S : s.B; }
bool no_rows(const at::Tensor &input) { return input.numel() == 0; }

at::Tensor state_or_zeros(const OptTensor &state, at::IntArrayRef shape, const at::TensorOptions &options) {
  return state.has_value() ? state->clone(at::MemoryFormat::Contiguous) : at::zeros(shape, options);
}

OptTensor contiguous(const OptTensor &t) { return t.has_value() ? OptTensor(t->contiguous()) : OptTensor(); }

struct Conv1d {
  dwconv_b200_sequence s;
  int taps;
  std::vector<int64_t> state;
};

Conv1d check_conv1d(const char *fn, const at::Tensor &input, const at::Tensor &weight, const OptTensor &bias,
                    const OptTensor &initial, const OptTensor &offsets) {
  Conv1d c;
  c.s = check_sequences(fn, input, offsets);
  TORCH_CHECK(weight.dim() == 3 && weight.size(0) == c.s.C && weight.size(1) == 1 && weight.size(2) >= 1 &&
                  weight.size(2) <= DWCONV_B200_MAX_TAPS,
              "dwconv_b200.", fn, ": weight must be [C, 1, taps] with C = ", c.s.C, " and 1 to ", DWCONV_B200_MAX_TAPS,
              " taps, got ", shape_text(weight));
  c.taps = (int)weight.size(2);
  check_operand(fn, "weight", weight, weight.sizes(), input.scalar_type(), input);
  if (bias.has_value()) check_operand(fn, "bias", *bias, {c.s.C}, input.scalar_type(), input);
  c.state = {state_count(c.s), c.taps - 1, c.s.C};
  if (initial.has_value()) check_operand(fn, "initial_state", *initial, c.state, input.scalar_type(), input);
  return c;
}

std::tuple<at::Tensor, OptTensor> conv1d_causal(const at::Tensor &input, const at::Tensor &weight,
                                                const OptTensor &bias, int64_t act, const OptTensor &initial,
                                                const OptTensor &offsets, bool want_state) {
  const char *fn = "depthwise_conv1d_causal";
  const Conv1d c = check_conv1d(fn, input, weight, bias, initial, offsets);
  c10::cuda::CUDAGuard guard(input.device());
  at::Tensor y = at::empty(input.sizes(), input.options(), at::MemoryFormat::Contiguous);
  OptTensor state;
  if (no_rows(input)) {
    if (want_state) state = state_or_zeros(initial, c.state, input.options());
    return {y, state};
  }
  if (want_state) state = at::empty(c.state, input.options());
  const at::Tensor x = rows_of(input), w = weight.contiguous();
  const OptTensor b = contiguous(bias), init = contiguous(initial);
  const dwconv_b200_rows xr = rows_arg(x);
  check_status(dwconv_b200_conv1d_causal(&xr, w.data_ptr(), ptr(b), ptr(init), y.data_ptr(),
                                         state.has_value() ? state->data_ptr() : nullptr, sequence_dtype(x), &c.s,
                                         c.taps, (int)act, stream_of(x)),
               fn);
  return {y, state};
}

// gradients of input, weight, bias, initial state (the last two: as asked)
std::tuple<at::Tensor, at::Tensor, OptTensor, OptTensor> conv1d_causal_backward(
    const at::Tensor &input, const at::Tensor &weight, const OptTensor &bias, int64_t act, const OptTensor &initial,
    const OptTensor &offsets, const OptTensor &grad, const OptTensor &grad_state, bool want_initial) {
  const char *fn = "depthwise_conv1d_causal backward";
  const Conv1d c = check_conv1d(fn, input, weight, bias, initial, offsets);
  c10::cuda::CUDAGuard guard(input.device());
  if (grad.has_value()) check_operand(fn, "grad_output", *grad, input.sizes(), input.scalar_type(), input);
  if (grad_state.has_value()) check_operand(fn, "grad_state", *grad_state, c.state, input.scalar_type(), input);
  OptTensor db, dinit;
  if (no_rows(input)) {
    if (bias.has_value()) db = at::zeros(bias->sizes(), input.options());
    if (want_initial) dinit = state_or_zeros(grad_state, c.state, input.options());
    return {at::empty(input.sizes(), input.options()), at::zeros(weight.sizes(), input.options()), db, dinit};
  }
  at::Tensor dx = at::empty(input.sizes(), input.options(), at::MemoryFormat::Contiguous);
  at::Tensor dw = at::empty(weight.sizes(), input.options(), at::MemoryFormat::Contiguous);
  if (bias.has_value()) db = at::empty({c.s.C}, input.options());
  if (want_initial) dinit = at::empty(c.state, input.options());
  const at::Tensor x = rows_of(input), w = weight.contiguous();
  const at::Tensor g = grad.has_value() ? rows_of(*grad) : at::zeros(input.sizes(), input.options());
  const OptTensor b = contiguous(bias), init = contiguous(initial), gs = contiguous(grad_state);
  const int code = sequence_dtype(x);
  const size_t nbytes = dwconv_b200_conv1d_causal_workspace_bytes(code, &c.s, c.taps);
  TORCH_CHECK(nbytes != 0, "dwconv_b200.", fn, ": invalid geometry");
  at::Tensor ws = at::empty({(int64_t)nbytes}, input.options().dtype(at::kByte));
  const dwconv_b200_rows xr = rows_arg(x), gr = rows_arg(g);
  check_status(dwconv_b200_conv1d_causal_backward(
                   &xr, w.data_ptr(), ptr(b), ptr(init), &gr, ptr(gs), dx.data_ptr(), dw.data_ptr(),
                   db.has_value() ? db->data_ptr() : nullptr, dinit.has_value() ? dinit->data_ptr() : nullptr,
                   ws.data_ptr(), nbytes, code, &c.s, c.taps, (int)act, stream_of(x)),
               fn);
  return {dx, dw, db, dinit};
}

// A state that a step updates in place.
void check_state(const char *fn, const at::Tensor &state, at::IntArrayRef shape, at::ScalarType type,
                 const at::Tensor &input) {
  check_operand(fn, "state", state, shape, type, input);
  TORCH_CHECK(state.is_contiguous(), "dwconv_b200.", fn, ": state is updated in place and must be contiguous");
}

// The kernels write through raw pointers: a graph that saved this state must learn of it.
void note_written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int64_t check_step_input(const char *fn, const at::Tensor &input) {
  check_cuda(input, "input");
  sequence_dtype(input);
  TORCH_CHECK(input.dim() == 2, "dwconv_b200.", fn, ": expected input [B, C], got ", shape_text(input));
  for (int d = 0; d < 2; ++d)
    TORCH_CHECK(input.size(d) <= (1ll << 30), "dwconv_b200.", fn, ": input is too large: ", shape_text(input));
  return input.size(1);
}

at::Tensor conv1d_causal_step(const at::Tensor &input, const at::Tensor &weight, const at::Tensor &state,
                              const OptTensor &bias, int64_t act) {
  const char *fn = "depthwise_conv1d_causal_step";
  const int64_t C = check_step_input(fn, input), B = input.size(0);
  TORCH_CHECK(weight.dim() == 3 && weight.size(0) == C && weight.size(1) == 1 && weight.size(2) >= 1 &&
                  weight.size(2) <= DWCONV_B200_MAX_TAPS,
              "dwconv_b200.", fn, ": weight must be [C, 1, taps] with C = ", C, " and 1 to ", DWCONV_B200_MAX_TAPS,
              " taps, got ", shape_text(weight));
  check_operand(fn, "weight", weight, weight.sizes(), input.scalar_type(), input);
  if (bias.has_value()) check_operand(fn, "bias", *bias, {C}, input.scalar_type(), input);
  const int taps = (int)weight.size(2);
  check_state(fn, state, {B, taps - 1, C}, input.scalar_type(), input);
  c10::cuda::CUDAGuard guard(input.device());
  at::Tensor y = at::empty({B, C}, input.options());
  if (no_rows(input)) return y;
  note_written(state);
  const at::Tensor x = rows_of(input), w = weight.contiguous();
  const OptTensor b = contiguous(bias);
  check_status(dwconv_b200_conv1d_causal_step(x.data_ptr(), x.stride(0), w.data_ptr(), ptr(b), state.data_ptr(),
                                              y.data_ptr(), sequence_dtype(x), (int)B, (int)C, taps, (int)act,
                                              stream_of(x)),
               fn);
  return y;
}

struct Recurrence {
  dwconv_b200_sequence s;
  std::vector<int64_t> state;
};

Recurrence check_recurrence(const char *fn, const at::Tensor &input, const at::Tensor &u, const at::Tensor &v,
                            const at::Tensor &decay, const OptTensor &initial, const OptTensor &offsets, double scale) {
  Recurrence r;
  r.s = check_sequences(fn, input, offsets);
  check_operand(fn, "recurrence_gate", u, input.sizes(), input.scalar_type(), input);
  check_operand(fn, "input_gate", v, input.sizes(), input.scalar_type(), input);
  check_operand(fn, "decay", decay, {r.s.C}, at::kFloat, input);
  r.state = {state_count(r.s), r.s.C};
  if (initial.has_value()) check_operand(fn, "initial_state", *initial, r.state, at::kFloat, input);
  TORCH_CHECK(scale > 0, "dwconv_b200.", fn, ": scale must be positive");
  return r;
}

// (y, final state or None, what the backward starts from or None)
std::tuple<at::Tensor, OptTensor, OptTensor> recurrence(const at::Tensor &input, const at::Tensor &gate_u,
                                                        const at::Tensor &gate_v, const at::Tensor &decay,
                                                        const OptTensor &initial, const OptTensor &offsets,
                                                        double scale, bool want_state, bool want_backward) {
  const char *fn = "gated_linear_recurrence";
  const Recurrence r = check_recurrence(fn, input, gate_u, gate_v, decay, initial, offsets, scale);
  c10::cuda::CUDAGuard guard(input.device());
  at::Tensor y = at::empty(input.sizes(), input.options(), at::MemoryFormat::Contiguous);
  const auto wide = input.options().dtype(at::kFloat);
  OptTensor state, ckpt;
  if (no_rows(input)) {
    if (want_state) state = state_or_zeros(initial, r.state, wide);
    if (want_backward) ckpt = at::empty({0}, wide);
    return {y, state, ckpt};
  }
  if (want_state) state = at::empty(r.state, wide);
  if (want_backward) {
    const size_t nbytes = dwconv_b200_recurrence_checkpoint_bytes(&r.s);
    TORCH_CHECK(nbytes != 0, "dwconv_b200.", fn, ": invalid geometry");
    ckpt = at::empty({(int64_t)(nbytes / 4)}, wide);
  }
  const at::Tensor x = rows_of(input), u = rows_of(gate_u), v = rows_of(gate_v), d = decay.contiguous();
  const OptTensor init = contiguous(initial);
  const dwconv_b200_rows xr = rows_arg(x), ur = rows_arg(u), vr = rows_arg(v);
  check_status(dwconv_b200_recurrence(&xr, &ur, &vr, d.data_ptr<float>(), (const float *)ptr(init), y.data_ptr(),
                                      state.has_value() ? state->data_ptr<float>() : nullptr,
                                      ckpt.has_value() ? ckpt->data_ptr<float>() : nullptr, sequence_dtype(x), &r.s,
                                      (float)scale, stream_of(x)),
               fn);
  return {y, state, ckpt};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, OptTensor> recurrence_backward(
    const at::Tensor &input, const at::Tensor &gate_u, const at::Tensor &gate_v, const at::Tensor &decay,
    const OptTensor &initial, const OptTensor &offsets, double scale, const at::Tensor &ckpt, const OptTensor &grad,
    const OptTensor &grad_state, bool want_initial) {
  const char *fn = "gated_linear_recurrence backward";
  const Recurrence r = check_recurrence(fn, input, gate_u, gate_v, decay, initial, offsets, scale);
  c10::cuda::CUDAGuard guard(input.device());
  if (grad.has_value()) check_operand(fn, "grad_output", *grad, input.sizes(), input.scalar_type(), input);
  if (grad_state.has_value()) check_operand(fn, "grad_state", *grad_state, r.state, at::kFloat, input);
  const auto wide = input.options().dtype(at::kFloat);
  at::Tensor dx = at::empty(input.sizes(), input.options(), at::MemoryFormat::Contiguous);
  at::Tensor du = at::empty_like(dx), dv = at::empty_like(dx);
  OptTensor dinit;
  if (no_rows(input)) {
    if (want_initial) dinit = state_or_zeros(grad_state, r.state, wide);
    return {dx, du, dv, at::zeros(decay.sizes(), wide), dinit};
  }
  check_kept(fn, "checkpoints", ckpt, {(int64_t)(dwconv_b200_recurrence_checkpoint_bytes(&r.s) / 4)}, input);
  at::Tensor dd = at::empty(decay.sizes(), wide);
  if (want_initial) dinit = at::empty(r.state, wide);
  const at::Tensor x = rows_of(input), u = rows_of(gate_u), v = rows_of(gate_v), d = decay.contiguous();
  const at::Tensor g = grad.has_value() ? rows_of(*grad) : at::zeros(input.sizes(), input.options());
  const OptTensor init = contiguous(initial), gs = contiguous(grad_state);
  const size_t nbytes = dwconv_b200_recurrence_workspace_bytes(&r.s);
  TORCH_CHECK(nbytes != 0, "dwconv_b200.", fn, ": invalid geometry");
  at::Tensor ws = at::empty({(int64_t)nbytes}, input.options().dtype(at::kByte));
  const dwconv_b200_rows xr = rows_arg(x), ur = rows_arg(u), vr = rows_arg(v), gr = rows_arg(g);
  check_status(dwconv_b200_recurrence_backward(
                   &xr, &ur, &vr, d.data_ptr<float>(), (const float *)ptr(init), ckpt.data_ptr<float>(), &gr,
                   (const float *)ptr(gs), dx.data_ptr(), du.data_ptr(), dv.data_ptr(), dd.data_ptr<float>(),
                   dinit.has_value() ? dinit->data_ptr<float>() : nullptr, ws.data_ptr(), nbytes, sequence_dtype(x),
                   &r.s, (float)scale, stream_of(x)),
               fn);
  return {dx, du, dv, dd, dinit};
}

at::Tensor recurrence_step(const at::Tensor &input, const at::Tensor &gate_u, const at::Tensor &gate_v,
                           const at::Tensor &decay, const at::Tensor &state, double scale) {
  const char *fn = "gated_linear_recurrence_step";
  const int64_t C = check_step_input(fn, input), B = input.size(0);
  check_operand(fn, "recurrence_gate", gate_u, input.sizes(), input.scalar_type(), input);
  check_operand(fn, "input_gate", gate_v, input.sizes(), input.scalar_type(), input);
  check_operand(fn, "decay", decay, {C}, at::kFloat, input);
  check_state(fn, state, {B, C}, at::kFloat, input);
  TORCH_CHECK(scale > 0, "dwconv_b200.", fn, ": scale must be positive");
  c10::cuda::CUDAGuard guard(input.device());
  at::Tensor y = at::empty({B, C}, input.options());
  if (no_rows(input)) return y;
  note_written(state);
  const at::Tensor x = rows_of(input), u = rows_of(gate_u), v = rows_of(gate_v), d = decay.contiguous();
  check_status(dwconv_b200_recurrence_step(x.data_ptr(), x.stride(0), u.data_ptr(), u.stride(0), v.data_ptr(),
                                           v.stride(0), d.data_ptr<float>(), state.data_ptr<float>(), y.data_ptr(),
                                           sequence_dtype(x), (int)B, (int)C, (float)scale, stream_of(x)),
               fn);
  return y;
}

// The rows of a tensor of any rank over its last dimension, as they lie where one stride steps
// through them, else as a contiguous copy.
at::Tensor norm_rows(const at::Tensor &t) {
  const int64_t C = t.size(-1);
  const at::Tensor a = rows_of(t);
  if (a.dim() == 2) return a;
  if (a.dim() == 1) return a.unsqueeze(0);
  int64_t stride = 0, span = 1;  // stride of the rows, and what the next outer dimension must step by
  bool ok = true, any = false;
  for (int64_t d = a.dim() - 2; d >= 0 && ok; --d) {
    if (a.size(d) == 1) continue;
    if (!any) {
      any = true;
      stride = a.stride(d);
    } else {
      ok = a.stride(d) == stride * span;
    }
    span *= a.size(d);
  }
  if (!ok) return a.contiguous().view({-1, C});
  return a.as_strided({span, C}, {any ? stride : C, 1}, a.storage_offset());
}

int64_t check_norm(const char *fn, const at::Tensor &input, const OptTensor &weight, const OptTensor &bias, double eps) {
  check_cuda(input, "input");
  sequence_dtype(input);
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) >= 1 && input.size(-1) <= (1 << 26), "dwconv_b200.", fn,
              ": expected input [..., C], got ", shape_text(input));
  const int64_t C = input.size(-1);
  if (weight.has_value()) check_operand(fn, "weight", *weight, {C}, input.scalar_type(), input);
  if (bias.has_value()) check_operand(fn, "bias", *bias, {C}, input.scalar_type(), input);
  TORCH_CHECK(eps >= 0, "dwconv_b200.", fn, ": eps must not be negative");
  return C;
}

// (y, (mean, rstd) of each row or None)
std::tuple<at::Tensor, OptTensor> layer_norm(const at::Tensor &input, const OptTensor &weight, const OptTensor &bias,
                                             double eps, bool want_backward) {
  const char *fn = "layer_norm";
  const int64_t C = check_norm(fn, input, weight, bias, eps), rows = input.numel() / C;
  c10::cuda::CUDAGuard guard(input.device());
  at::Tensor y = at::empty(input.sizes(), input.options(), at::MemoryFormat::Contiguous);
  OptTensor stats;
  if (want_backward) stats = at::empty({rows, 2}, input.options().dtype(at::kFloat));
  if (rows == 0) return {y, stats};
  const at::Tensor x = norm_rows(input);
  const OptTensor w = contiguous(weight), b = contiguous(bias);
  check_status(dwconv_b200_layer_norm(x.data_ptr(), x.stride(0), ptr(w), ptr(b), y.data_ptr(),
                                      stats.has_value() ? stats->data_ptr<float>() : nullptr, sequence_dtype(x), rows,
                                      (int)C, (float)eps, stream_of(x)),
               fn);
  return {y, stats};
}

std::tuple<at::Tensor, OptTensor, OptTensor> layer_norm_backward(const at::Tensor &input, const OptTensor &weight,
                                                                 const at::Tensor &stats, const at::Tensor &grad,
                                                                 bool want_weight, bool want_bias) {
  const char *fn = "layer_norm backward";
  const int64_t C = check_norm(fn, input, weight, OptTensor(), 0.), rows = input.numel() / C;
  check_operand(fn, "grad_output", grad, input.sizes(), input.scalar_type(), input);
  c10::cuda::CUDAGuard guard(input.device());
  at::Tensor dx = at::empty(input.sizes(), input.options(), at::MemoryFormat::Contiguous);
  OptTensor dw, db, ws;
  if (rows == 0) {
    if (want_weight) dw = at::zeros({C}, input.options());
    if (want_bias) db = at::zeros({C}, input.options());
    return {dx, dw, db};
  }
  check_kept(fn, "stats", stats, {rows, 2}, input);
  if (want_weight) dw = at::empty({C}, input.options());
  if (want_bias) db = at::empty({C}, input.options());
  const at::Tensor x = norm_rows(input), g = norm_rows(grad);
  const OptTensor w = contiguous(weight);
  const int code = sequence_dtype(x);
  size_t nbytes = 0;
  if (want_weight || want_bias) {
    nbytes = dwconv_b200_layer_norm_workspace_bytes(code, rows, (int)C);
    TORCH_CHECK(nbytes != 0, "dwconv_b200.", fn, ": invalid geometry");
    ws = at::empty({(int64_t)nbytes}, input.options().dtype(at::kByte));
  }
  check_status(dwconv_b200_layer_norm_backward(
                   x.data_ptr(), x.stride(0), ptr(w), stats.data_ptr<float>(), g.data_ptr(), g.stride(0), dx.data_ptr(),
                   dw.has_value() ? dw->data_ptr() : nullptr, db.has_value() ? db->data_ptr() : nullptr,
                   ws.has_value() ? ws->data_ptr() : nullptr, nbytes, code, rows, (int)C, stream_of(x)),
               fn);
  return {dx, dw, db};
}

// ---- autograd nodes ---------------------------------------------------------------------
// What the Python functions call: checks, the forward call and, where something wants a gradient, a node
// of the autograd graph, without a trip through the interpreter in either direction.  Gradients are
// first-order only (the message is the one of torch.autograd.function.once_differentiable).

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

at::Tensor or_undefined(const OptTensor &t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor or_none(const at::Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

template <typename... T> bool wants_grad(const T &...t) {
  return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

// There are no forward-mode derivatives: a tangent that an operand carries would be lost.
template <typename... T> void refuse_tangents(const char *fn, const T &...t) {
  TORCH_CHECK(!(torch::autograd::isFwGradDefined(t) || ...), "dwconv_b200.", fn,
              ": forward-mode differentiation is not supported");
}

struct OnceNode : torch::autograd::Node {
  // A leaf's gradient is accumulated on the stream that was current when a live graph first reached the
  // leaf.  Where that is the legacy default stream, which cannot take part in a capture, the engine would
  // break the capture in the middle; refused here, before anything is recorded.  Leaves behind views and conversions
  // (parameters under autocast) count like those that the node reads itself.
  void check_capture() {
    const at::DeviceIndex device = this->device().index();
    const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream(device);
    if (current.id() == 0) return;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(current.stream(), &status) != cudaSuccess || status == cudaStreamCaptureStatusNone)
      return;
    const auto *info = torch::autograd::get_current_graph_task_exec_info();  // empty: every node runs
    std::vector<torch::autograd::Node *> todo{this};
    std::unordered_set<torch::autograd::Node *> seen;
    while (!todo.empty()) {
      const torch::autograd::Node *n = todo.back();
      todo.pop_back();
      for (const torch::autograd::Edge &edge : n->next_edges()) {
        torch::autograd::Node *fn = edge.function.get();
        if (fn == nullptr || !seen.insert(fn).second) continue;
        if (info != nullptr && !info->empty()) {
          const auto at = info->find(fn);
          if (at == info->end() || !at->second.should_execute()) continue;
        }
        if (dynamic_cast<torch::autograd::AccumulateGrad *>(fn) == nullptr) {
          todo.push_back(fn);
          continue;
        }
        const auto stream = fn->stream();
        TORCH_CHECK(!stream.has_value() || stream->id() != 0, "dwconv_b200: ", name(),
                    " is being captured into a CUDA graph, but an eager autograd graph of the same leaf is still alive "
                    "on the default stream; release it before the capture");
      }
    }
  }
  variable_list apply(variable_list &&grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    check_capture();
    bool any = false;
    for (const at::Tensor &g : grads) any = any || g.defined();
    variable_list out(num_outputs());
    if (!any) return out;
    {
      at::AutoGradMode no_grad(false);
      backward(grads, out);
    }
    // with create_graph: the gradients depend on the inputs even where those that came in are constants
    if (at::GradMode::is_enabled()) {
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)out.size());
      for (at::Tensor &t : out)
        if (t.defined()) t = t.detach().requires_grad_(true);
      out = (*error)(std::move(out));
    }
    return out;
  }
  virtual void backward(const variable_list &grads, variable_list &out) = 0;
  at::Tensor saved(SavedVariable &v) { return v.unpack(shared_from_this()); }
  OptTensor saved_or_none(SavedVariable &v) { return or_none(v.unpack(shared_from_this())); }
};

template <typename N, typename... T> std::shared_ptr<N> new_node(const T &...inputs) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  n->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return n;
}

struct CausalConv1dNode : OnceNode {
  SavedVariable input, weight, bias, initial, offsets;
  int64_t act;
  std::string name() const override { return "CausalConv1dBackward"; }
  void release_variables() override {
    for (SavedVariable *v : {&input, &weight, &bias, &initial, &offsets}) v->reset_data();
  }
  void backward(const variable_list &grads, variable_list &out) override {
    auto [dx, dw, db, dinit] = conv1d_causal_backward(
        saved(input), saved(weight), saved_or_none(bias), act, saved_or_none(initial), saved_or_none(offsets),
        or_none(grads[0]), grads.size() > 1 ? or_none(grads[1]) : OptTensor(), task_should_compute_output(3));
    out[0] = dx;
    out[1] = dw;
    out[2] = or_undefined(db);
    out[3] = or_undefined(dinit);
  }
};

py::object conv1d_causal_autograd(const at::Tensor &input, const at::Tensor &weight, const OptTensor &bias, int64_t act,
                                  const OptTensor &initial, const OptTensor &offsets, bool want_state) {
  const at::Tensor b = or_undefined(bias), h = or_undefined(initial);
  at::Tensor y;
  OptTensor state;
  refuse_tangents("depthwise_conv1d_causal", input, weight, b, h);
  const bool grad = wants_grad(input, weight, b, h);
  {
    at::AutoGradMode no_grad(false);
    std::tie(y, state) = conv1d_causal(input, weight, bias, act, initial, offsets, want_state);
  }
  if (grad) {
    auto n = new_node<CausalConv1dNode>(input, weight, b, h);
    n->input = SavedVariable(input, false);
    n->weight = SavedVariable(weight, false);
    n->bias = SavedVariable(b, false);
    n->initial = SavedVariable(h, false);
    n->offsets = SavedVariable(or_undefined(offsets), false);
    n->act = act;
    torch::autograd::set_history(y, n);
    if (want_state) torch::autograd::set_history(*state, n);
  }
  if (want_state) return py::make_tuple(y, *state);
  return py::cast(y);
}

struct RecurrenceNode : OnceNode {
  SavedVariable input, u, v, decay, initial, offsets, ckpt;
  double scale;
  std::string name() const override { return "GatedLinearRecurrenceBackward"; }
  void release_variables() override {
    for (SavedVariable *s : {&input, &u, &v, &decay, &initial, &offsets, &ckpt}) s->reset_data();
  }
  void backward(const variable_list &grads, variable_list &out) override {
    auto [dx, du, dv, dd, dinit] = recurrence_backward(
        saved(input), saved(u), saved(v), saved(decay), saved_or_none(initial), saved_or_none(offsets), scale,
        saved(ckpt), or_none(grads[0]), grads.size() > 1 ? or_none(grads[1]) : OptTensor(), task_should_compute_output(4));
    out[0] = dx;
    out[1] = du;
    out[2] = dv;
    out[3] = dd;
    out[4] = or_undefined(dinit);
  }
};

py::object recurrence_autograd(const at::Tensor &input, const at::Tensor &u, const at::Tensor &v,
                               const at::Tensor &decay, const OptTensor &initial, const OptTensor &offsets,
                               double scale, bool want_state) {
  const at::Tensor h = or_undefined(initial);
  at::Tensor y;
  OptTensor state, ckpt;
  refuse_tangents("gated_linear_recurrence", input, u, v, decay, h);
  const bool grad = wants_grad(input, u, v, decay, h);
  {
    at::AutoGradMode no_grad(false);
    std::tie(y, state, ckpt) = recurrence(input, u, v, decay, initial, offsets, scale, want_state, grad);
  }
  if (grad) {
    auto n = new_node<RecurrenceNode>(input, u, v, decay, h);
    n->input = SavedVariable(input, false);
    n->u = SavedVariable(u, false);
    n->v = SavedVariable(v, false);
    n->decay = SavedVariable(decay, false);
    n->initial = SavedVariable(h, false);
    n->offsets = SavedVariable(or_undefined(offsets), false);
    n->ckpt = SavedVariable(*ckpt, false);
    n->scale = scale;
    torch::autograd::set_history(y, n);
    if (want_state) torch::autograd::set_history(*state, n);
  }
  if (want_state) return py::make_tuple(y, *state);
  return py::cast(y);
}

struct LayerNormNode : OnceNode {
  SavedVariable input, weight, stats;
  std::string name() const override { return "ChannelLayerNormBackward"; }
  void release_variables() override {
    for (SavedVariable *s : {&input, &weight, &stats}) s->reset_data();
  }
  void backward(const variable_list &grads, variable_list &out) override {
    auto [dx, dw, db] = layer_norm_backward(saved(input), saved_or_none(weight), saved(stats), grads[0],
                                            task_should_compute_output(1), task_should_compute_output(2));
    out[0] = dx;
    out[1] = or_undefined(dw);
    out[2] = or_undefined(db);
  }
};

at::Tensor layer_norm_autograd(const at::Tensor &input, const OptTensor &weight, const OptTensor &bias, double eps) {
  const at::Tensor w = or_undefined(weight), b = or_undefined(bias);
  at::Tensor y;
  OptTensor stats;
  refuse_tangents("layer_norm", input, w, b);
  const bool grad = wants_grad(input, w, b);
  {
    at::AutoGradMode no_grad(false);
    std::tie(y, stats) = layer_norm(input, weight, bias, eps, grad);
  }
  if (grad) {
    auto n = new_node<LayerNormNode>(input, w, b);
    n->input = SavedVariable(input, false);
    n->weight = SavedVariable(w, false);
    n->stats = SavedVariable(*stats, false);
    torch::autograd::set_history(y, n);
  }
  return y;
}

// The steps have no gradient: what would want one is refused.
at::Tensor conv1d_causal_step_checked(const at::Tensor &input, const at::Tensor &weight, const at::Tensor &state,
                                      const OptTensor &bias, int64_t act) {
  TORCH_CHECK(!wants_grad(input, weight, state, or_undefined(bias)),
              "dwconv_b200.depthwise_conv1d_causal_step: the state is updated in place and has no gradient; use "
              "depthwise_conv1d_causal or torch.no_grad()");
  refuse_tangents("depthwise_conv1d_causal_step", input, weight, state, or_undefined(bias));
  return conv1d_causal_step(input, weight, state, bias, act);
}

at::Tensor recurrence_step_checked(const at::Tensor &input, const at::Tensor &u, const at::Tensor &v,
                                   const at::Tensor &decay, const at::Tensor &state, double scale) {
  TORCH_CHECK(!wants_grad(input, u, v, decay, state),
              "dwconv_b200.gated_linear_recurrence_step: the state is updated in place and has no gradient; use "
              "gated_linear_recurrence or torch.no_grad()");
  refuse_tangents("gated_linear_recurrence_step", input, u, v, decay, state);
  return recurrence_step(input, u, v, decay, state, scale);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "dwconv_b200 tensor-level binding (links libdwconv_b200.so)";
  m.def("library_version", []() { return dwconv_b200_version(); });
  m.def("forward", &forward);
  m.def("backward", &backward);
  m.def("use_dwconv2d_small", &use_dwconv2d_small);
  m.def("dwconv2d", &dwconv2d);
  m.def("dwconv2d_small", &dwconv2d_small);
  m.def("dwconv2d_backward_kernel", &dwconv2d_backward_kernel);
  m.def("conv1d_causal", &conv1d_causal);
  m.def("conv1d_causal_backward", &conv1d_causal_backward);
  m.def("conv1d_causal_step", &conv1d_causal_step);
  m.def("recurrence", &recurrence);
  m.def("recurrence_backward", &recurrence_backward);
  m.def("recurrence_step", &recurrence_step);
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("conv1d_causal_autograd", &conv1d_causal_autograd);
  m.def("conv1d_causal_step_checked", &conv1d_causal_step_checked);
  m.def("recurrence_autograd", &recurrence_autograd);
  m.def("recurrence_step_checked", &recurrence_step_checked);
  m.def("layer_norm_autograd", &layer_norm_autograd);
}
