// Causal depthwise convolution of [B, T, C] sequences, its gradients and its one-row step
// (declarations: include/dwconv_b200.h).
//
//   p[t] = bias + sum_k w[k] x[t - (K-1) + k],  y = act(p)
//   dp = dy act'(p),  dx[t] = sum_k w[k] dp[t + K-1-k],  dw[k] = sum_t dp[t] x[t - (K-1) + k],  db = sum_t dp[t]
//
// Bound by memory (forward: x in, y out; backward: x and dy in, dx out).  A warp owns 32 * V channels
// and a run of R rows; the rows stream through a register window, so each is read once, but for the
// K-1 rows in front of a run (backward: behind it too), which come from L1 / L2.  The sums are in fp32.
//
// Packed sequences: a warp's row number is the same in all lanes, so a sequence's end is one uniform
// comparison per row; there the window is filled anew from the next sequence's initial rows.
#include <initializer_list>

#include "seq_common.cuh"

namespace dwb {
namespace {

constexpr int CONV_WARPS = 8;

struct Conv1dParams {
  SeqList q;
  int R;           // rows of a run
  int cblocks;     // channel blocks
  int rblocks;     // blocks of CONV_WARPS runs per batch element
  long long main;  // CTAs that walk rows; those behind them fill the states
  int act;
};

__device__ __forceinline__ float2 act2(float2 p, int act) {
  if (act == DWCONV_B200_ACT_NONE) return p;
  if (act == DWCONV_B200_ACT_SILU) return mul2(p, sigmoid2(p));
  return make_float2(apply_activation<float>(p.x, act), apply_activation<float>(p.y, act));
}

__device__ __forceinline__ float slope(float p, int act) {
  switch (act) {
    case DWCONV_B200_ACT_RELU: return p > 0.f ? 1.f : 0.f;
    case DWCONV_B200_ACT_RELU6: return p > 0.f && p < 6.f ? 1.f : 0.f;
    case DWCONV_B200_ACT_HARDSWISH: return p <= -3.f ? 0.f : (p >= 3.f ? 1.f : (2.f * p + 3.f) / 6.f);
    default: return 1.f;
  }
}
// g act'(p)
__device__ __forceinline__ float2 act_back2(float2 g, float2 p, int act) {
  if (act == DWCONV_B200_ACT_NONE) return g;
  if (act == DWCONV_B200_ACT_SILU) {
    const float2 s = sigmoid2(p);
    return mul2(mul2(g, s), fma2(p, one_minus2(s), f2(1.f)));
  }
  return mul2(g, make_float2(slope(p.x, act), slope(p.y, act)));
}

__device__ __forceinline__ SeqSpan conv_span(const SeqList &q, int b, int t) {
  if (q.offsets != nullptr) return seq_locate(q, t);
  return SeqSpan{b, 0, q.T};
}

// The K-1 rows in front of row t, oldest first: rows of the sequence, or of its initial state.
template <typename T, int H, bool VEC, int K>
__device__ __forceinline__ void fill_window(float2 (&win)[K][H], const Lanes<T, H, VEC> &ln, const SeqIn<T> &x,
                                            const T *initial, int C, int b, int t, const SeqSpan &sp) {
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int row = t - (K - 1) + j;
    typename Lanes<T, H, VEC>::Raw raw = ln.zero();
    if (row >= sp.begin) raw = ln.load(x.row(b, row));
    else if (initial != nullptr && sp.seq >= 0)
      raw = ln.load(initial + ((long long)sp.seq * (K - 1) + (row - sp.begin + K - 1)) * C);
    ln.get(raw, win[j]);
  }
}

template <int H, int K> __device__ __forceinline__ void shift(float2 (&a)[K][H]) {
#pragma unroll
  for (int k = 0; k + 1 < K; ++k)
#pragma unroll
    for (int h = 0; h < H; ++h) a[k][h] = a[k + 1][h];
}

// The taps (and bias) of a lane's channels.
template <typename T, int H, bool VEC, int K> struct Taps {
  float2 w[K][H], b[H];
  __device__ __forceinline__ Taps(const Lanes<T, H, VEC> &ln, const T *wt, const T *bias) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int c = ln.channel(2 * h), d = ln.channel(2 * h + 1);
#pragma unroll
      for (int k = 0; k < K; ++k)
        w[k][h] = make_float2(read(wt + (long long)c * K + k), read(wt + (long long)d * K + k));
      b[h] = bias != nullptr ? make_float2(read(bias + c), read(bias + d)) : f2(0.f);
    }
  }
  // the sum over a window, taps in order
  __device__ __forceinline__ void apply(const float2 (&win)[K][H], float2 (&o)[H]) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      o[h] = b[h];
#pragma unroll
      for (int k = 0; k < K; ++k) o[h] = fma2(w[k][h], win[k][h], o[h]);
    }
  }
};

// The last K-1 rows of each sequence.
template <typename T, int K>
__device__ void final_rows(const SeqIn<T> &x, const T *initial, T *fin, const SeqList &q, int part, int parts) {
  const long long n = (long long)q.S * (K - 1) * q.C;
  for (long long i = (long long)part * blockDim.x + threadIdx.x; i < n; i += (long long)parts * blockDim.x) {
    const int c = (int)(i % q.C);
    const long long jr = i / q.C;
    const int r = (int)(jr % (K - 1)), j = (int)(jr / (K - 1));
    int s = 0, e = q.T;
    if (q.offsets) {
      s = seq_bound(q, j);
      e = max(s, seq_bound(q, j + 1));
    }
    const int row = e - (K - 1) + r;
    T v = Elem<T>::from_acc(0.f);
    if (row >= s) v = x.row(q.offsets ? 0 : j, row)[c];
    else if (initial) v = initial[((long long)j * (K - 1) + (row - s + K - 1)) * q.C + c];
    fin[i] = v;
  }
}

template <typename T, int H, bool VEC, int K>
__global__ void __launch_bounds__(CONV_WARPS * 32, K <= 4 ? 3 : 2)
conv1d_forward_kernel(SeqIn<T> x, const T *__restrict__ w, const T *__restrict__ bias, const T *__restrict__ initial,
                      T *__restrict__ y, T *__restrict__ fin, Conv1dParams p) {
  using Ln = Lanes<T, H, VEC>;
  constexpr int U = sizeof(T) == 4 ? 4 : 8;  // rows loaded together
  if (blockIdx.x >= p.main) {
    if constexpr (K > 1) final_rows<T, K>(x, initial, fin, p.q, (int)(blockIdx.x - p.main), (int)(gridDim.x - p.main));
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  const int cb = (int)(blockIdx.x % p.cblocks);
  const long long rest = blockIdx.x / p.cblocks;
  const int rb = (int)(rest % p.rblocks), b = (int)(rest / p.rblocks);
  const int C = p.q.C;
  const long long first = ((long long)rb * CONV_WARPS + warp) * p.R;
  if (first >= p.q.T) return;
  const int t0 = (int)first, t1 = min(t0 + p.R, p.q.T);
  const Ln ln(cb, threadIdx.x & 31, C);
  const Taps<T, H, VEC, K> taps(ln, w, bias);
  SeqSpan sp = conv_span(p.q, b, t0);
  float2 win[K][H];
  fill_window(win, ln, x, initial, C, b, t0, sp);
  int t = t0;
  while (t < t1) {
    if (t == sp.next) {
      sp = conv_span(p.q, b, t);
      fill_window(win, ln, x, initial, C, b, t, sp);
    }
    const T *xr = x.row(b, t);
    T *yr = y + ((long long)b * p.q.T + t) * C;
    if (t + U <= t1 && t + U <= sp.next && sp.seq >= 0) {
      typename Ln::Raw raw[U];
#pragma unroll
      for (int j = 0; j < U; ++j) raw[j] = ln.load(xr + j * x.rs);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float2 o[H];
        ln.get(raw[j], win[K - 1]);
        taps.apply(win, o);
#pragma unroll
        for (int h = 0; h < H; ++h) o[h] = act2(o[h], p.act);
        ln.store(yr + (long long)j * C, o);
        shift(win);
      }
      t += U;
    } else {
      float2 o[H];
      ln.get(ln.load(xr), win[K - 1]);
      taps.apply(win, o);
#pragma unroll
      for (int h = 0; h < H; ++h) o[h] = sp.seq >= 0 ? act2(o[h], p.act) : f2(0.f);
      ln.store(yr, o);
      shift(win);
      ++t;
    }
  }
}

// dx, the initial rows' gradient, and this CTA's part of dw and db: part[block of runs][K + 1][C].
template <typename T, int H, bool VEC, int K>
__global__ void __launch_bounds__(CONV_WARPS * 32, 2)
conv1d_backward_kernel(SeqIn<T> x, const T *__restrict__ w, const T *__restrict__ bias, const T *__restrict__ initial,
                       SeqIn<T> dy, const T *__restrict__ dfin, T *__restrict__ dx, T *__restrict__ dinit,
                       float *__restrict__ part, Conv1dParams p) {
  using Ln = Lanes<T, H, VEC>;
  if (blockIdx.x >= p.main) {  // sequences without a row: their state passes through
    const long long each = (long long)(K - 1) * p.q.C;
    for (int j = (int)(blockIdx.x - p.main); j < p.q.S; j += (int)(gridDim.x - p.main)) {
      const int s = p.q.offsets ? seq_bound(p.q, j) : 0, e = p.q.offsets ? seq_bound(p.q, j + 1) : p.q.T;
      if (e > s) continue;
      for (long long i = threadIdx.x; i < each; i += blockDim.x)
        dinit[j * each + i] = dfin ? dfin[j * each + i] : Elem<T>::from_acc(0.f);
    }
    return;
  }
  __shared__ float2 sum[(K + 1) * H][32];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  const int cb = (int)(blockIdx.x % p.cblocks);
  const long long rest = blockIdx.x / p.cblocks;
  const int rb = (int)(rest % p.rblocks), b = (int)(rest / p.rblocks);
  const int C = p.q.C;
  const Ln ln(cb, lane, C);
  const long long first = ((long long)rb * CONV_WARPS + warp) * p.R;
  float2 dwk[K][H], db[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    db[h] = f2(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) dwk[k][h] = f2(0.f);
  }
  if (first < p.q.T) {
    const int t0 = (int)first, t1 = min(t0 + p.R, p.q.T);
    const Taps<T, H, VEC, K> taps(ln, w, bias);
    float2 win[K][H], dpw[K][H];  // rows t-(K-1) .. t of x and of dp, oldest first; t's place is free between rows
    SeqSpan sp = conv_span(p.q, b, t0);
    fill_window(win, ln, x, initial, C, b, t0, sp);
    auto clear = [&]() {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int h = 0; h < H; ++h) dpw[k][h] = f2(0.f);
    };
    clear();
    // the gradient of row t - (K-1), complete once dp[t] is in the window (oldest dp: tap K-1)
    auto gradient = [&](float2 (&o)[H]) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        o[h] = mul2(taps.w[0][h], dpw[K - 1][h]);
#pragma unroll
        for (int k = 1; k < K; ++k) o[h] = fma2(taps.w[k][h], dpw[K - 1 - k][h], o[h]);
      }
    };
    // a row's gradient to where it belongs: dx, or the initial rows of a sequence that starts here
    auto emit = [&](int row, const float2 (&o)[H]) {
      if (row >= sp.begin) {
        if (row >= t0 && row < t1) ln.store(dx + ((long long)b * p.q.T + row) * C, o);
      } else if (dinit != nullptr && sp.seq >= 0 && sp.begin >= t0 && sp.begin < t1) {
        ln.store(dinit + ((long long)sp.seq * (K - 1) + (row - sp.begin + K - 1)) * C, o);
      }
    };
    auto take = [&](const typename Ln::Raw &rx, const typename Ln::Raw &rg) {
      float2 g[H], s[H];
      ln.get(rx, win[K - 1]);
      ln.get(rg, g);
      taps.apply(win, s);
#pragma unroll
      for (int h = 0; h < H; ++h) dpw[K - 1][h] = act_back2(g[h], s[h], p.act);
    };
    auto count = [&]() {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        db[h] = add2(db[h], dpw[K - 1][h]);
#pragma unroll
        for (int k = 0; k < K; ++k) dwk[k][h] = fma2(dpw[K - 1][h], win[k][h], dwk[k][h]);
      }
    };

    constexpr int U = 4;
    int t = t0;
    while (true) {
      if (t >= t1 + K - 1) break;
      if (t == sp.next) {
        // the sequence ends: its last K-1 rows take no more products, but are its final state
#pragma unroll
        for (int f = 0; f < K - 1; ++f) {
          float2 o[H];
#pragma unroll
          for (int h = 0; h < H; ++h) dpw[K - 1][h] = f2(0.f);
          gradient(o);
          if (dfin != nullptr && sp.seq >= 0) {
            float2 d[H];
            ln.get(ln.load(dfin + ((long long)sp.seq * (K - 1) + f) * C), d);
#pragma unroll
            for (int h = 0; h < H; ++h) o[h] = add2(o[h], d[h]);
          }
          emit(t + f - (K - 1), o);
          shift(dpw);
        }
        if (t >= t1) break;
        sp = conv_span(p.q, b, t);
        fill_window(win, ln, x, initial, C, b, t, sp);
        clear();
      }
      const int lead = t - (K - 1);
      if (lead >= t0 && lead >= sp.begin && t + U <= t1 && t + U <= sp.next && sp.seq >= 0) {
        // U rows inside the run and the sequence
        typename Ln::Raw rx[U], rg[U];
        const T *xr = x.row(b, t), *gr = dy.row(b, t);
        T *dr = dx + ((long long)b * p.q.T + lead) * C;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          rx[j] = ln.load(xr + j * x.rs);
          rg[j] = ln.load(gr + j * dy.rs);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
          float2 o[H];
          take(rx[j], rg[j]);
          count();
          gradient(o);
          ln.store(dr + (long long)j * C, o);
          shift(win);
          shift(dpw);
        }
        t += U;
      } else {
        typename Ln::Raw rx = ln.zero(), rg = ln.zero();
        if (sp.seq >= 0) {
          rx = ln.load(x.row(b, t));
          rg = ln.load(dy.row(b, t));
        }
        take(rx, rg);
        if (sp.seq < 0) {
#pragma unroll
          for (int h = 0; h < H; ++h) dpw[K - 1][h] = f2(0.f);
        } else if (t < t1) {
          count();
        }
        float2 o[H];
        gradient(o);
        emit(lead, o);
        shift(win);
        shift(dpw);
        ++t;
      }
    }
  }
  for (int n = 0; n < CONV_WARPS; ++n) {  // warp after warp, in order
    if (warp == n) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int m = 0; m <= K; ++m) {
          float2 *s = &sum[m * H + h][lane];
          const float2 v = m < K ? dwk[m < K ? m : 0][h] : db[h];
          *s = n ? add2(*s, v) : v;
        }
      }
    }
    __syncthreads();
  }
  float *mine = part + rest * (K + 1) * C;
  for (int m = threadIdx.x; m < (K + 1) * Ln::GROUP; m += blockDim.x) {  // consecutive threads, consecutive channels
    const int n = m % Ln::GROUP, k = m / Ln::GROUP, ch = cb * Ln::GROUP + n;
    const int l = VEC ? n / (2 * H) : n % 32, i = VEC ? n % (2 * H) : n / 32;
    const float2 v = sum[k * H + i / 2][l];
    if (ch < C) mine[(long long)k * C + ch] = i & 1 ? v.y : v.x;
  }
}

template <typename T, int H, bool VEC, int K>
__global__ void __launch_bounds__(128)
conv1d_step_kernel(const T *__restrict__ x, long long xs, const T *__restrict__ w, const T *__restrict__ bias,
                   T *__restrict__ state, T *__restrict__ y, long long units, int groups, int C, int act) {
  using Ln = Lanes<T, H, VEC>;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);  // a group of channels of a batch element
  if (unit >= units) return;
  const Ln ln((int)(unit % groups), threadIdx.x & 31, C);
  const long long b = unit / groups;
  T *st = state + b * (K - 1) * C;
  typename Ln::Raw raw[K];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) raw[k] = ln.load(st + (long long)k * C);
  raw[K - 1] = ln.load(x + b * xs);
  const Taps<T, H, VEC, K> taps(ln, w, bias);
  float2 win[K][H], o[H];
#pragma unroll
  for (int k = 0; k < K; ++k) ln.get(raw[k], win[k]);
  taps.apply(win, o);
#pragma unroll
  for (int h = 0; h < H; ++h) o[h] = act2(o[h], act);
  ln.store(y + b * C, o);
  __syncwarp();  // lanes that share channels have all read their state
#pragma unroll
  for (int k = 0; k < K - 1; ++k) ln.store(st + (long long)k * C, win[k + 1]);
}

// ---- host --------------------------------------------------------------------------------------

// Rows of a run: as many as leave about 16 warps per SM (a longer run re-reads fewer rows in front of
// it), between 8 and 64.  Counted for 128 channels per warp whatever the variant, so that the size of
// the workspace follows from the problem alone.
inline int conv_run(int B, int T, int C) {
  const long long per_row = (long long)B * ceil_div(C, 128);
  int R = 64;
  while (R > 8 && per_row * ceil_div(T, R) < 148 * 16) R >>= 1;
  return R;
}

inline Conv1dParams conv_params(const dwconv_b200_sequence &s, int group, int act) {
  Conv1dParams p;
  p.q = seq_list(s);
  p.R = conv_run(s.B, s.T, s.C);
  p.cblocks = ceil_div(s.C, group);
  p.rblocks = ceil_div(ceil_div(s.T, p.R), CONV_WARPS);
  p.main = (long long)p.cblocks * p.rblocks * s.B;
  p.act = act;
  return p;
}

inline long long conv_parts(const dwconv_b200_sequence &s) {
  return (long long)ceil_div(ceil_div(s.T, conv_run(s.B, s.T, s.C)), CONV_WARPS) * s.B;
}

constexpr int STATE_BLOCKS = 64;  // most CTAs that fill the states

#define DWB_TAPS(K, CALL)                                        \
  switch (K) {                                                   \
    case 1: { constexpr int TAPS = 1; CALL; } break;             \
    case 2: { constexpr int TAPS = 2; CALL; } break;             \
    case 3: { constexpr int TAPS = 3; CALL; } break;             \
    case 4: { constexpr int TAPS = 4; CALL; } break;             \
    case 5: { constexpr int TAPS = 5; CALL; } break;             \
    case 6: { constexpr int TAPS = 6; CALL; } break;             \
    case 7: { constexpr int TAPS = 7; CALL; } break;             \
    default: { constexpr int TAPS = 8; CALL; } break;            \
  }

struct ConvArgs {
  const dwconv_b200_rows *x, *dy;
  const void *w, *bias, *initial, *dfin;
  void *y, *fin, *dx, *dinit;
  float *part;
  const dwconv_b200_sequence *s;
  int taps, act;
};

template <typename T, int H, bool VEC> void launch_forward(const ConvArgs &a, cudaStream_t st) {
  const Conv1dParams p = conv_params(*a.s, Lanes<T, H, VEC>::GROUP, a.act);
  long long extra = 0;
  if (a.fin != nullptr && a.taps > 1) {
    extra = ceil_div_ll((long long)p.q.S * (a.taps - 1) * p.q.C, CONV_WARPS * 32);
    if (extra > STATE_BLOCKS) extra = STATE_BLOCKS;
  }
  if (p.main + extra == 0) return;
  DWB_TAPS(a.taps, (conv1d_forward_kernel<T, H, VEC, TAPS><<<(unsigned)(p.main + extra), CONV_WARPS * 32, 0, st>>>(
                       seq_in<T>(*a.x), (const T *)a.w, (const T *)a.bias, (const T *)a.initial, (T *)a.y,
                       (T *)a.fin, p)))
}

// Register windows of x, dp, w and dw: four channels per lane for up to four taps, two above.
template <typename T, int H, bool VEC> void launch_backward(const ConvArgs &a, cudaStream_t st) {
  const Conv1dParams p = conv_params(*a.s, a.taps > 4 ? 64 : Lanes<T, H, VEC>::GROUP, a.act);
  long long extra = 0;
  if (a.dinit != nullptr && a.taps > 1 && (a.s->offsets != nullptr || a.s->T == 0))
    extra = p.q.S < STATE_BLOCKS ? p.q.S : STATE_BLOCKS;
  if (p.main + extra == 0) return;
  DWB_TAPS(a.taps, (conv1d_backward_kernel<T, (TAPS > 4 ? 1 : H), VEC, TAPS>
                    <<<(unsigned)(p.main + extra), CONV_WARPS * 32, 0, st>>>(
                        seq_in<T>(*a.x), (const T *)a.w, (const T *)a.bias, (const T *)a.initial, seq_in<T>(*a.dy),
                        (const T *)a.dfin, (T *)a.dx, (T *)a.dinit, a.part, p)))
}

// Whether everything that moves V channels at a time may.
inline bool conv_vector(const ConvArgs &a, int V, size_t es) {
  const void *ptrs[] = {a.initial, a.dfin, a.y, a.dx, a.dinit};
  for (const void *q : ptrs)
    if (q != nullptr && !aligned_to(q, V * es)) return false;
  return a.s->C % V == 0 && rows_vector(*a.x, V, es) && (a.dy == nullptr || rows_vector(*a.dy, V, es));
}

template <typename T> void forward_t(const ConvArgs &a, cudaStream_t st) {
  if (conv_vector(a, 4, sizeof(T))) launch_forward<T, 2, true>(a, st);
  else launch_forward<T, 1, false>(a, st);
}
template <typename T> void backward_t(const ConvArgs &a, cudaStream_t st) {
  if (conv_vector(a, 4, sizeof(T))) launch_backward<T, 2, true>(a, st);
  else launch_backward<T, 1, false>(a, st);
}

template <typename T, int H, bool VEC>
void launch_step(const void *x, long long xs, const void *w, const void *bias, void *state, void *y, int B, int C,
                 int taps, int act, cudaStream_t st) {
  const int groups = ceil_div(C, Lanes<T, H, VEC>::GROUP);
  const long long units = (long long)B * groups;
  const unsigned grid = (unsigned)ceil_div_ll(units, 4);
  DWB_TAPS(taps, (conv1d_step_kernel<T, H, VEC, TAPS><<<grid, 128, 0, st>>>(
                     (const T *)x, xs, (const T *)w, (const T *)bias, (T *)state, (T *)y, units, groups, C, act)))
}

template <typename T>
void step_t(const void *x, long long xs, const void *w, const void *bias, void *state, void *y, int B, int C,
            int taps, int act, cudaStream_t st) {
  if (C % 4 == 0 && xs % 4 == 0 && aligned_to(x, 4 * sizeof(T)) && aligned_to(state, 4 * sizeof(T)) &&
      aligned_to(y, 4 * sizeof(T)))
    launch_step<T, 2, true>(x, xs, w, bias, state, y, B, C, taps, act, st);
  else
    launch_step<T, 1, false>(x, xs, w, bias, state, y, B, C, taps, act, st);
}

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
    case DWCONV_B200_F32: forward_t<float>(a, st); break;
    case DWCONV_B200_F16: forward_t<__half>(a, st); break;
    default: forward_t<__nv_bfloat16>(a, st); break;
  }
  return api_launch_status();
}

size_t dwconv_b200_conv1d_causal_workspace_bytes(int dtype, const dwconv_b200_sequence *seq, int taps) {
  if (check_conv(dtype, seq, taps) != DWCONV_B200_OK) return 0;
  const size_t n = (size_t)conv_parts(*seq) * (taps + 1) * seq->C * sizeof(float);
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
  switch (dtype) {
    case DWCONV_B200_F32: backward_t<float>(a, st); break;
    case DWCONV_B200_F16: backward_t<__half>(a, st); break;
    default: backward_t<__nv_bfloat16>(a, st); break;
  }
  e = api_launch_status();
  if (e) return e;
  launch_column_sum(a.part, conv_parts(*seq), (taps + 1) * seq->C,
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
    case DWCONV_B200_F32: step_t<float>(x, x_stride, w, bias, state, y, B, C, taps, activation, st); break;
    case DWCONV_B200_F16: step_t<__half>(x, x_stride, w, bias, state, y, B, C, taps, activation, st); break;
    default: step_t<__nv_bfloat16>(x, x_stride, w, bias, state, y, B, C, taps, activation, st); break;
  }
  return api_launch_status();
}

}  // extern "C"
