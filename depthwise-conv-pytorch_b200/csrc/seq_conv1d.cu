// Causal depthwise convolution of sequences: entry points (declarations: include/dwconv_b200.h).
#include <initializer_list>

#include "seq_conv1d_ops.cuh"

namespace dwb {
namespace {

int check_conv(int dtype, const dwconv_b200_sequence *s, int taps) {
  if (!seq_dtype_ok(dtype)) return DWCONV_B200_UNSUPPORTED_DTYPE;
  const int e = check_sequence(s);
  if (e) return e;
  if (taps < 1) return DWCONV_B200_BAD_ARGUMENT;
  if (taps > DWCONV_B200_MAX_TAPS) return DWCONV_B200_UNSUPPORTED_SHAPE;
  // one CTA per (channel block, block of runs, batch element)
  if ((long long)ceil_div(s->C, 32) * ceil_div(ceil_div(s->T, 8), CONV_WARPS) * s->B > (1ll << 31) - 1 - STATE_BLOCKS)
    return DWCONV_B200_TOO_LARGE;
  return DWCONV_B200_OK;
}

inline bool act_ok(int act) { return act >= DWCONV_B200_ACT_NONE && act <= DWCONV_B200_ACT_HARDSWISH; }

inline bool all_aligned(std::initializer_list<const void *> ptrs, size_t a) {
  for (const void *p : ptrs)
    if (p != nullptr && !aligned_to(p, a)) return false;
  return true;
}

}  // namespace
}  // namespace dwb

using namespace dwb;

extern "C" {

int dwconv_b200_conv1d_causal(const dwconv_b200_rows *x, const void *w, const void *bias, const void *initial,
                              void *y, void *final_state, int dtype, const dwconv_b200_sequence *seq, int taps,
                              int activation, void *stream) {
  int e = check_conv(dtype, seq, taps);
  if (e) return e;
  const size_t es = elem_size(dtype);
  if ((e = check_rows(x, es)) != 0) return e;
  if (w == nullptr || y == nullptr || !act_ok(activation)) return DWCONV_B200_BAD_ARGUMENT;
  if (!all_aligned({w, bias, initial, y, final_state}, es)) return DWCONV_B200_MISALIGNED;
  ConvArgs a{};
  a.x = x; a.w = w; a.bias = bias; a.initial = initial; a.y = y; a.fin = final_state;
  a.s = seq; a.taps = taps; a.act = activation;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: conv1d_forward<float>(a, st); break;
    case DWCONV_B200_F16: conv1d_forward<__half>(a, st); break;
    default: conv1d_forward<__nv_bfloat16>(a, st); break;
  }
  return api_launch_status();
}

size_t dwconv_b200_conv1d_causal_workspace_bytes(int dtype, const dwconv_b200_sequence *seq, int taps) {
  if (check_conv(dtype, seq, taps) != DWCONV_B200_OK) return 0;
  // for whichever variant the pointers' alignment will allow
  long long parts = 0;
  for (int group : {64, 128}) {
    const Conv1dParams p = conv_params(*seq, group, 0, true);
    if ((long long)p.rblocks * seq->B > parts) parts = (long long)p.rblocks * seq->B;
  }
  const size_t n = (size_t)parts * (taps + 1) * seq->C * sizeof(float);
  return (n + 15) / 16 * 16 + 16;
}

int dwconv_b200_conv1d_causal_backward(const dwconv_b200_rows *x, const void *w, const void *bias,
                                       const void *initial, const dwconv_b200_rows *dy, const void *dfinal,
                                       void *dx, void *dw, void *dbias, void *dinitial, void *workspace,
                                       size_t workspace_bytes, int dtype, const dwconv_b200_sequence *seq,
                                       int taps, int activation, void *stream) {
  int e = check_conv(dtype, seq, taps);
  if (e) return e;
  const size_t es = elem_size(dtype);
  if ((e = check_rows(x, es)) != 0 || (e = check_rows(dy, es)) != 0) return e;
  if (w == nullptr || dx == nullptr || dw == nullptr || workspace == nullptr || !act_ok(activation))
    return DWCONV_B200_BAD_ARGUMENT;
  if (!all_aligned({w, bias, initial, dfinal, dx, dw, dbias, dinitial}, es) || !aligned_to(workspace, 16))
    return DWCONV_B200_MISALIGNED;
  if (workspace_bytes < dwconv_b200_conv1d_causal_workspace_bytes(dtype, seq, taps))
    return DWCONV_B200_WORKSPACE_TOO_SMALL;
  ConvArgs a{};
  a.x = x; a.w = w; a.bias = bias; a.initial = initial; a.dy = dy; a.dfin = dfinal; a.dx = dx; a.dinit = dinitial;
  a.part = static_cast<float *>(workspace);
  a.s = seq; a.taps = taps; a.act = activation;
  cudaStream_t st = (cudaStream_t)stream;
  long long parts = 0;
  switch (dtype) {
    case DWCONV_B200_F32: parts = conv1d_backward<float>(a, st); break;
    case DWCONV_B200_F16: parts = conv1d_backward<__half>(a, st); break;
    default: parts = conv1d_backward<__nv_bfloat16>(a, st); break;
  }
  e = api_launch_status();
  if (e) return e;
  launch_column_sum(a.part, parts, (taps + 1) * seq->C,
                    ColumnSumOut{dw, dbias, dtype, seq->C, taps, nullptr}, st);
  return api_launch_status();
}

int dwconv_b200_conv1d_causal_step(const void *x, long long x_stride, const void *w, const void *bias, void *state,
                                   void *y, int dtype, int B, int C, int taps, int activation, void *stream) {
  const dwconv_b200_sequence s{B, 1, C, nullptr, 0};
  const int e = check_conv(dtype, &s, taps);
  if (e) return e;
  if (x == nullptr || w == nullptr || y == nullptr || (state == nullptr && taps > 1) || !act_ok(activation))
    return DWCONV_B200_BAD_ARGUMENT;
  const size_t es = elem_size(dtype);
  if (!all_aligned({x, w, bias, state, y}, es)) return DWCONV_B200_MISALIGNED;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: conv1d_step<float>(x, x_stride, w, bias, state, y, B, C, taps, activation, st); break;
    case DWCONV_B200_F16: conv1d_step<__half>(x, x_stride, w, bias, state, y, B, C, taps, activation, st); break;
    default: conv1d_step<__nv_bfloat16>(x, x_stride, w, bias, state, y, B, C, taps, activation, st); break;
  }
  return api_launch_status();
}

}  // extern "C"
