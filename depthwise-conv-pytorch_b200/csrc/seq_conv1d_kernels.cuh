// Causal depthwise convolution of [B, T, C] sequences, its gradients and its one-row step:
// kernels and launches.
//
//   p[t] = bias + sum_k w[k] x[t - (K-1) + k],  y = act(p)
//   dp = dy act'(p),  dx[t] = sum_k w[k] dp[t + K-1-k],  dw[k] = sum_t dp[t] x[t - (K-1) + k],  db = sum_t dp[t]
//
// Bound by memory (forward: x in, y out; backward: x and dy in, dx out).  A warp owns 64 or 128
// channels and a run of R rows; the rows stream through a register window, so each is read once, but for the
// K-1 rows in front of a run (backward: behind it too), which come from L1 / L2.  The sums are in fp32.
// Rows are copied to shared memory some chunks of rows ahead (cp.async), every lane the bytes that it will
// read itself: no barrier, no registers for what is on its way.
//
// Measured (bf16, four taps, SiLU, 4 x 4096 rows of 2560 channels): forward 32 us, 5.3 TB/s (6.1 TB/s on 8 x 8192
// rows of 4096), backward 71 us, 3.5 TB/s (4.9): its windows and sums leave two CTAs per SM.  Odd widths, whose rows
// are loaded where they are used (2561 channels): 57 and 122 us.
//
// Packed sequences: a warp's row number is the same in all lanes, so a sequence's end is one uniform
// comparison per row; there the window is filled anew from the next sequence's initial rows.
#pragma once

#include <atomic>

#include "seq_conv1d_ops.cuh"

namespace dwb {
namespace {

// ACT: the two activations that have kernels of their own, or ANY with the activation at run time.
constexpr int ANY = -1;

// A NaN stays one, and passes the gradient on.
__device__ __forceinline__ float activate(float p, int act) {
  return act == DWCONV_B200_ACT_RELU ? (p <= 0.f ? 0.f : p) : apply_activation<float>(p, act);
}
template <int ACT> __device__ __forceinline__ float2 act2(float2 p, int act) {
  if constexpr (ACT == DWCONV_B200_ACT_NONE) return p;
  if constexpr (ACT == DWCONV_B200_ACT_SILU) return mul2(p, sigmoid2(p));
  return make_float2(activate(p.x, act), activate(p.y, act));
}

__device__ __forceinline__ float slope(float p, int act) {
  switch (act) {
    case DWCONV_B200_ACT_RELU: return p <= 0.f ? 0.f : 1.f;
    case DWCONV_B200_ACT_RELU6: return p <= 0.f || p >= 6.f ? 0.f : 1.f;
    case DWCONV_B200_ACT_HARDSWISH: return p <= -3.f ? 0.f : (p >= 3.f ? 1.f : (2.f * p + 3.f) / 6.f);
    default: return 1.f;
  }
}
// g act'(p)
template <int ACT> __device__ __forceinline__ float2 act_back2(float2 g, float2 p, int act) {
  if constexpr (ACT == DWCONV_B200_ACT_NONE) return g;
  if constexpr (ACT == DWCONV_B200_ACT_SILU) {
    const float2 s = sigmoid2(p);
    return mul2(mul2(g, s), fma2(p, one_minus2(s), f2(1.f)));
  }
  return mul2(g, make_float2(slope(p.x, act), slope(p.y, act)));
}

__device__ __forceinline__ SeqSpan conv_span(const SeqList &q, int b, int t) {
  if (q.offsets != nullptr) return seq_locate(q, t);
  return SeqSpan{b, 0, q.T};
}

// A window of K rows is a ring: `at` is the place of its oldest row.  Loops unrolled by a multiple of K know
// it at compile time and end where they began, so that no row is moved.
template <int K> __host__ __device__ constexpr int ring(int at, int k) { return (at + k) % K; }
// Rows a lane loads together: a multiple of K.
template <int K> constexpr int conv_unroll(int most) { return K >= most ? K : most / K * K; }

// Chunks of U rows of NT tensors on their way to a lane: STAGES - 1 of them while one is worked on.
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
template <typename T, int H, int U, int NT> struct RowPipe {
  using Raw = typename Lanes<T, H, true>::Raw;
  static constexpr int CHUNK = U * NT * 32 * (int)sizeof(Raw);  // bytes of a warp's chunk
  static constexpr int FIT = 64 * 1024 / (CONV_WARPS * CHUNK);
  static constexpr int STAGES = FIT < 2 ? 2 : (FIT > 4 ? 4 : FIT);
  static constexpr int BYTES = CONV_WARPS * STAGES * CHUNK;     // of a CTA
  const unsigned char *mine;
  __device__ __forceinline__ RowPipe(unsigned char *smem, int warp, int lane)
      : mine(smem + warp * STAGES * CHUNK + lane * (int)sizeof(Raw)) {}
  __device__ __forceinline__ const Raw *at(int stage, int j, int n) const {
    return reinterpret_cast<const Raw *>(mine + stage * CHUNK + (j * NT + n) * 32 * (int)sizeof(Raw));
  }
  // row[n]: this lane's place in the chunk's first row of tensor n, rs[n] elements between rows
  __device__ __forceinline__ void start(int stage, const T *const (&row)[NT], const long long (&rs)[NT]) const {
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        copy_async<(int)sizeof(Raw)>((uint32_t)__cvta_generic_to_shared(at(stage, j, n)), row[n] + j * rs[n]);
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // the oldest of the chunks on their way has arrived
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }
  // `chunks` chunks from the given rows on: body(chunk, stage) once chunk has arrived.
  template <typename F>
  __device__ __forceinline__ void run(int chunks, const T *const (&first)[NT], const long long (&rs)[NT], F &&body) const {
    const T *row[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) row[n] = first[n];
    auto next = [&](int i, int stage) {
      if (i < chunks) {
        start(stage, row, rs);
#pragma unroll
        for (int n = 0; n < NT; ++n) row[n] += U * rs[n];
      }
      commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) next(i, i);
    int stage = 0;
    for (int i = 0; i < chunks; ++i) {
      wait();
      body(i, stage);
      next(i + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
  }
};
template <typename T, int H, bool VEC, int U, int NT> constexpr int pipe_bytes() {
  if constexpr (VEC) return RowPipe<T, H, U, NT>::BYTES;
  else return 0;
}
template <typename T, int K> constexpr int forward_unroll() { return conv_unroll<K>(4); }

// The K-1 rows in front of row t, oldest first at 0: rows of the sequence, or of its initial state.
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

// The oldest row gives its place up, outside the unrolled loops: the rest move to the front.
template <int H, int K> __device__ __forceinline__ void shift(float2 (&a)[K][H]) {
#pragma unroll
  for (int k = 0; k + 1 < K; ++k)
#pragma unroll
    for (int h = 0; h < H; ++h) a[k][h] = a[k + 1][h];
}

// The taps (and bias) of a lane's channels.  Those of adjacent channels are adjacent: K loads of as many
// values as the lane has channels (their address is a multiple of that many values, so aligned where the
// filter is).
template <typename T, int H, bool VEC, int K> struct Taps {
  float2 w[K][H], b[H];
  __device__ __forceinline__ Taps(const Lanes<T, H, VEC> &ln, const T *wt, const T *bias) {
    float f[2 * H][K];
    if constexpr (VEC) {
      using P = Pack<T, 2 * H>;
      float q[K][2 * H];
#pragma unroll
      for (int n = 0; n < K; ++n) P::unpack(P::load(wt + (long long)ln.channel(0) * K + n * 2 * H), q[n]);
#pragma unroll
      for (int i = 0; i < 2 * H; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k) f[i][k] = q[(i * K + k) / (2 * H)][(i * K + k) % (2 * H)];
    } else {
#pragma unroll
      for (int i = 0; i < 2 * H; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k) f[i][k] = read(wt + (long long)ln.channel(i) * K + k);
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][h] = make_float2(f[2 * h][k], f[2 * h + 1][k]);
      b[h] = bias != nullptr ? make_float2(read(bias + ln.channel(2 * h)), read(bias + ln.channel(2 * h + 1))) : f2(0.f);
    }
  }
  // the sum over a window, taps in order
  __device__ __forceinline__ void apply(const float2 (&win)[K][H], int at, float2 (&o)[H]) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      o[h] = b[h];
#pragma unroll
      for (int k = 0; k < K; ++k) o[h] = fma2(w[k][h], win[ring<K>(at, k)][h], o[h]);
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

template <typename T, int H, bool VEC, int K, int ACT>
__global__ void __launch_bounds__(CONV_WARPS * 32, K <= 4 ? 3 : 2)
conv1d_forward_kernel(SeqIn<T> x, const T *__restrict__ w, const T *__restrict__ bias, const T *__restrict__ initial,
                      T *__restrict__ y, T *__restrict__ fin, Conv1dParams p) {
  using Ln = Lanes<T, H, VEC>;
  constexpr int U = forward_unroll<T, K>();
  extern __shared__ __align__(16) unsigned char pipe_smem[];
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
    const int chunks = sp.seq >= 0 ? (min(t1, sp.next) - t) / U : 0;
    if (chunks > 0) {
      auto rows = [&](const typename Ln::Raw (&raw)[U], T *out) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
          float2 o[H];
          ln.get(raw[j], win[ring<K>(j, K - 1)]);
          taps.apply(win, j, o);
#pragma unroll
          for (int h = 0; h < H; ++h) o[h] = act2<ACT>(o[h], p.act);
          ln.store(out + (long long)j * C, o);
        }
      };
      if constexpr (VEC) {
        const RowPipe<T, H, U, 1> pipe(pipe_smem, warp, threadIdx.x & 31);
        pipe.run(chunks, {xr + ln.channel(0)}, {x.rs}, [&](int i, int stage) {
          typename Ln::Raw raw[U];
#pragma unroll
          for (int j = 0; j < U; ++j) raw[j] = *pipe.at(stage, j, 0);
          rows(raw, yr + (long long)i * U * C);
        });
      } else {
        for (int i = 0; i < chunks; ++i) {
          typename Ln::Raw raw[U];
#pragma unroll
          for (int j = 0; j < U; ++j) raw[j] = ln.load(xr + ((long long)i * U + j) * x.rs);
          rows(raw, yr + (long long)i * U * C);
        }
      }
      t += chunks * U;
    } else {
      float2 o[H];
      ln.get(ln.load(xr), win[K - 1]);
      taps.apply(win, 0, o);
#pragma unroll
      for (int h = 0; h < H; ++h) o[h] = sp.seq >= 0 ? act2<ACT>(o[h], p.act) : f2(0.f);
      ln.store(yr, o);
      shift(win);
      ++t;
    }
  }
}

// dx, the initial rows' gradient, and this CTA's part of dw and db: part[block of runs][K + 1][C].
template <typename T, int H, bool VEC, int K, int ACT>
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
  extern __shared__ __align__(16) unsigned char pipe_smem[];
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
    float2 win[K][H], dpw[K][H];  // rows t-(K-1) .. t of x and of dp; t's place is free between rows
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
    auto gradient = [&](int at, float2 (&o)[H]) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        o[h] = mul2(taps.w[0][h], dpw[ring<K>(at, K - 1)][h]);
#pragma unroll
        for (int k = 1; k < K; ++k) o[h] = fma2(taps.w[k][h], dpw[ring<K>(at, K - 1 - k)][h], o[h]);
      }
    };
    // the same outside the chunks, where rows of the window may lie outside the sequence: taps lo .. hi
    // alone (a tap times a zero is no zero where the tap is not finite)
    auto border_gradient = [&](int lo, int hi, float2 (&o)[H]) {
#pragma unroll
      for (int h = 0; h < H; ++h) o[h] = f2(0.f);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (k >= lo && k <= hi) {
#pragma unroll
          for (int h = 0; h < H; ++h) o[h] = fma2(taps.w[k][h], dpw[K - 1 - k][h], o[h]);
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
    auto take = [&](int at, const typename Ln::Raw &rx, const typename Ln::Raw &rg) {
      float2 g[H], s[H];
      ln.get(rx, win[ring<K>(at, K - 1)]);
      ln.get(rg, g);
      if constexpr (ACT != DWCONV_B200_ACT_NONE) taps.apply(win, at, s);
#pragma unroll
      for (int h = 0; h < H; ++h)
        dpw[ring<K>(at, K - 1)][h] = ACT == DWCONV_B200_ACT_NONE ? g[h] : act_back2<ACT>(g[h], s[h], p.act);
    };
    auto count = [&](int at) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float2 d = dpw[ring<K>(at, K - 1)][h];
        db[h] = add2(db[h], d);
#pragma unroll
        for (int k = 0; k < K; ++k) dwk[k][h] = fma2(d, win[ring<K>(at, k)][h], dwk[k][h]);
      }
    };

    constexpr int U = conv_unroll<K>(4);
    int t = t0;
    while (true) {
      if (t >= t1 + K - 1) break;
      if (t == sp.next) {
        // the sequence ends: its last K-1 rows take no more products, but are its final state
#pragma unroll
        for (int f = 0; f < K - 1; ++f) {
          float2 o[H];
          border_gradient(f + 1, sp.seq >= 0 ? t + f - sp.begin : -1, o);
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
      const int chunks = lead >= t0 && lead >= sp.begin && sp.seq >= 0 ? (min(t1, sp.next) - t) / U : 0;
      if (chunks > 0) {
        // chunks of U rows inside the run and the sequence
        const T *xr = x.row(b, t), *gr = dy.row(b, t);
        T *dr = dx + ((long long)b * p.q.T + lead) * C;
        auto row = [&](int j, const typename Ln::Raw &rx, const typename Ln::Raw &rg, T *out) {
          float2 o[H];
          take(j, rx, rg);
          count(j);
          gradient(j, o);
          ln.store(out, o);
        };
        if constexpr (VEC) {
          const RowPipe<T, H, U, 2> pipe(pipe_smem, warp, lane);
          pipe.run(chunks, {xr + ln.channel(0), gr + ln.channel(0)}, {x.rs, dy.rs}, [&](int i, int stage) {
            T *out = dr + (long long)i * U * C;
#pragma unroll
            for (int j = 0; j < U; ++j) row(j, *pipe.at(stage, j, 0), *pipe.at(stage, j, 1), out + (long long)j * C);
          });
        } else {
          for (int i = 0; i < chunks; ++i) {
            typename Ln::Raw rx[U], rg[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
              rx[j] = ln.load(xr + ((long long)i * U + j) * x.rs);
              rg[j] = ln.load(gr + ((long long)i * U + j) * dy.rs);
            }
            T *out = dr + (long long)i * U * C;
#pragma unroll
            for (int j = 0; j < U; ++j) row(j, rx[j], rg[j], out + (long long)j * C);
          }
        }
        t += chunks * U;
      } else {
        typename Ln::Raw rx = ln.zero(), rg = ln.zero();
        if (sp.seq >= 0) {
          rx = ln.load(x.row(b, t));
          rg = ln.load(dy.row(b, t));
        }
        take(0, rx, rg);
        if (sp.seq < 0) {
#pragma unroll
          for (int h = 0; h < H; ++h) dpw[K - 1][h] = f2(0.f);
        } else if (t < t1) {
          count(0);
        }
        float2 o[H];
        border_gradient(0, sp.seq >= 0 ? t - sp.begin : -1, o);
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
  taps.apply(win, 0, o);
#pragma unroll
  for (int h = 0; h < H; ++h)
    o[h] = act == DWCONV_B200_ACT_SILU ? act2<DWCONV_B200_ACT_SILU>(o[h], act) : act2<ANY>(o[h], act);
  ln.store(y + b * C, o);
  __syncwarp();  // lanes that share channels have all read their state
#pragma unroll
  for (int k = 0; k < K - 1; ++k) ln.store(st + (long long)k * C, win[k + 1]);
}

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

#define DWB_ACT(A, CALL)                                                                     \
  if ((A) == DWCONV_B200_ACT_NONE) { constexpr int ACT = DWCONV_B200_ACT_NONE; CALL; }       \
  else if ((A) == DWCONV_B200_ACT_SILU) { constexpr int ACT = DWCONV_B200_ACT_SILU; CALL; }  \
  else { constexpr int ACT = ANY; CALL; }


// One kernel with its shared memory; what that takes is set once per kernel and device.
template <auto KERNEL, int SMEM, typename... A> void launch_rows(long long ctas, cudaStream_t st, A... args) {
  static std::atomic<unsigned long long> ready{0};
  if (SMEM > 32 * 1024) {  // with the static part, more than 48 KB
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
      if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return;
      ready.fetch_or(bit, std::memory_order_release);
    }
  }
  KERNEL<<<(unsigned)ctas, CONV_WARPS * 32, SMEM, st>>>(args...);
}

template <typename T, int H, bool VEC> void launch_forward(const ConvArgs &a, cudaStream_t st) {
  const Conv1dParams p = conv_params(*a.s, Lanes<T, H, VEC>::GROUP, a.act, false);
  long long extra = 0;
  if (a.fin != nullptr && a.taps > 1) {
    extra = ceil_div_ll((long long)p.q.S * (a.taps - 1) * p.q.C, CONV_WARPS * 32);
    if (extra > STATE_BLOCKS) extra = STATE_BLOCKS;
  }
  if (p.main + extra == 0) return;
  DWB_TAPS(a.taps, DWB_ACT(a.act, (launch_rows<conv1d_forward_kernel<T, H, VEC, TAPS, ACT>,
                                               pipe_bytes<T, H, VEC, forward_unroll<T, TAPS>(), 1>()>(
                                      p.main + extra, st, seq_in<T>(*a.x), (const T *)a.w, (const T *)a.bias,
                                      (const T *)a.initial, (T *)a.y, (T *)a.fin, p))))
}

// Register windows of x, dp, w and dw: four channels per lane for up to four taps, two above.
// Returns the parts of the filter's gradient.
template <typename T, int H, bool VEC> long long launch_backward(const ConvArgs &a, cudaStream_t st) {
  const Conv1dParams p = conv_params(*a.s, a.taps > 4 ? 64 : Lanes<T, H, VEC>::GROUP, a.act, true);
  long long extra = 0;
  if (a.dinit != nullptr && a.taps > 1 && (a.s->offsets != nullptr || a.s->T == 0))
    extra = p.q.S < STATE_BLOCKS ? p.q.S : STATE_BLOCKS;
  if (p.main + extra == 0) return 0;
  DWB_TAPS(a.taps, DWB_ACT(a.act, (launch_rows<conv1d_backward_kernel<T, (TAPS > 4 ? 1 : H), VEC, TAPS, ACT>,
                                               pipe_bytes<T, (TAPS > 4 ? 1 : H), VEC, conv_unroll<TAPS>(4), 2>()>(
                                      p.main + extra, st, seq_in<T>(*a.x), (const T *)a.w, (const T *)a.bias,
                                      (const T *)a.initial, seq_in<T>(*a.dy), (const T *)a.dfin, (T *)a.dx,
                                      (T *)a.dinit, a.part, p))))
  return (long long)p.rblocks * a.s->B;
}

// Whether everything that moves V channels at a time may.
inline bool conv_vector(const ConvArgs &a, int V, size_t es) {
  const void *ptrs[] = {a.w, a.initial, a.dfin, a.y, a.dx, a.dinit};
  for (const void *q : ptrs)
    if (q != nullptr && !aligned_to(q, V * es)) return false;
  return a.s->C % V == 0 && rows_vector(*a.x, V, es) && (a.dy == nullptr || rows_vector(*a.dy, V, es));
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

}  // namespace

template <typename T> void conv1d_forward(const ConvArgs &a, cudaStream_t st) {
  if (conv_vector(a, 4, sizeof(T))) launch_forward<T, 2, true>(a, st);
  else launch_forward<T, 1, false>(a, st);
}
template <typename T> long long conv1d_backward(const ConvArgs &a, cudaStream_t st) {
  return conv_vector(a, 4, sizeof(T)) ? launch_backward<T, 2, true>(a, st) : launch_backward<T, 1, false>(a, st);
}

template <typename T>
void conv1d_step(const void *x, long long xs, const void *w, const void *bias, void *state, void *y, int B, int C,
            int taps, int act, cudaStream_t st) {
  if (C % 4 == 0 && xs % 4 == 0 && aligned_to(x, 4 * sizeof(T)) && aligned_to(w, 4 * sizeof(T)) && aligned_to(state, 4 * sizeof(T)) &&
      aligned_to(y, 4 * sizeof(T)))
    launch_step<T, 2, true>(x, xs, w, bias, state, y, B, C, taps, act, st);
  else
    launch_step<T, 1, false>(x, xs, w, bias, state, y, B, C, taps, act, st);
}

#define DWB_CONV1D_INSTANTIATE(T)                                                                                    \
  template void conv1d_forward<T>(const ConvArgs &, cudaStream_t);                                                   \
  template long long conv1d_backward<T>(const ConvArgs &, cudaStream_t);                                             \
  template void conv1d_step<T>(const void *, long long, const void *, const void *, void *, void *, int, int, int,   \
                               int, cudaStream_t);

}  // namespace dwb
