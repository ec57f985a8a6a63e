// What the translation units of the causal depthwise convolution share: its arguments, and how a
// problem is cut into runs of rows.
#pragma once

#include "seq_common.cuh"

namespace dwb {

constexpr int CONV_WARPS = 8;

struct Conv1dParams {
  SeqList q;
  int R;           // rows of a run
  int cblocks;     // channel blocks
  int rblocks;     // blocks of CONV_WARPS runs per batch element
  long long main;  // CTAs that walk rows; those behind them fill the states
  int act;
};

struct ConvArgs {
  const dwconv_b200_rows *x, *dy;
  const void *w, *bias, *initial, *dfin;
  void *y, *fin, *dx, *dinit;
  float *part;
  const dwconv_b200_sequence *s;
  int taps, act;
};

// Rows of a run: the choice whose rounds of resident CTAs (counted as three per SM forward, two backward), each a
// run and what it costs beside its rows, take least.  That cost is worth 5 rows forward (the filter, the K-1 rows
// in front) and 12 backward (those on both sides, the sums at the end).  Forward kernels of five taps and more
// are bounded to two CTAs per SM, which the count does not know.  Measured with runs of 16 / 24 / 32 / 48 / 64 / 128
// rows (microseconds, start included): 4 x 4096 rows of 2560 channels, bf16, four taps: forward 43 / 39 / 37 / 37 /
// 39 / 43 (it takes 48), backward 125 / 102 / 92 / 82 / 82 / 82 (48); 8 x 8192 rows of 4096: 215 / 193 / 182 / 178 /
// 172 / 176 (128), backward 707 / 557 / 475 / 410 / 373 / 332 (128); 2 x 8192 rows of 576, fp32, seven taps: 23 / 23 /
// 27 / 25 / 25 / 31 (24), backward 68 / 59 / 51 / 51 / 41 / 47 (64); 4099 rows of 1001, fp16: 18 / 14 / 16 / 18 / 21 /
// 33 (24), backward 31 / 35 / 25 / 29 / 33 / 47 (32).
inline int conv_run(const dwconv_b200_sequence &s, int group, bool backward) {
  static const int runs[] = {8, 16, 24, 32, 48, 64, 96, 128};
  const long long slots = 148 * (backward ? 2 : 3), per_block = (long long)s.B * ceil_div(s.C, group);
  int best = runs[0];
  long long cost = 0;
  for (int R : runs) {
    const long long ctas = per_block * ceil_div(ceil_div(s.T, R), CONV_WARPS);
    const long long c = ceil_div_ll(ctas, slots) * (R + (backward ? 12 : 5));
    if (R == runs[0] || c < cost) {
      best = R;
      cost = c;
    }
  }
  return best;
}

inline Conv1dParams conv_params(const dwconv_b200_sequence &s, int group, int act, bool backward) {
  Conv1dParams p;
  p.q = seq_list(s);
  p.R = conv_run(s, group, backward);
  p.cblocks = ceil_div(s.C, group);
  p.rblocks = ceil_div(ceil_div(s.T, p.R), CONV_WARPS);
  p.main = (long long)p.cblocks * p.rblocks * s.B;
  p.act = act;
  return p;
}

constexpr int STATE_BLOCKS = 64;  // most CTAs that fill the states

// One translation unit per element type (seq_conv1d_f32.cu, seq_conv1d_f16.cu, seq_conv1d_bf16.cu).
template <typename T> void conv1d_forward(const ConvArgs &a, cudaStream_t st);
// Returns the parts of the filter's gradient.
template <typename T> long long conv1d_backward(const ConvArgs &a, cudaStream_t st);
template <typename T>
void conv1d_step(const void *x, long long xs, const void *w, const void *bias, void *state, void *y, int B, int C,
                 int taps, int act, cudaStream_t st);

}  // namespace dwb
