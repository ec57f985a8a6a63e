// Layer norm over the channels of a row, forward and backward (declarations: include/dwconv_b200.h).
//
//   y = (x - m) s w + b,  m = mean, s = 1 / sqrt(mean (x - m)^2 + eps)
//   with xh = (x - m) s and q = dy w:   dx = s (q - mean(q) - xh mean(q xh)),
//   dw = sum over rows of dy xh,  db = sum over rows of dy.
//
// Bound by memory (forward: x in, y out; backward: x, dy in, dx out), which a row's two sums interrupt.  Both
// directions read each row once: `tpr` threads own a row (a power of two, up to 512) and keep its values
// in registers as they came, NV vectors of V elements per thread, and the next row is on its way
// meanwhile.  CTAs stay for many rows (backward: with w in registers).  The variance is the sum of
// squares around the mean (warps' sums are merged by the parallel-variance formula, so that one
// exchange through shared memory gives both moments), never a difference of large sums.
//
// Measured (bf16, 16384 rows of 4096): forward 59 us, 4.5 TB/s, bound by the issue of instructions (356 per warp
// and 512 values; 76 % of the slots); backward 83 us, 4.8 TB/s, one CTA of 512 threads per SM, whose
// registers hold the sums of dw and db.  fp32: 97 and 176 us (5.5 and 4.6 TB/s).  1001 bf16 values, one per load: 58
// and 54 us (1.1 and 1.8 TB/s); 8192 rows of 12288 bf16 values by the wide kernels: 245 and 415 us (1.6 and
// 1.5 TB/s).
#include "seq_common.cuh"

namespace dwb {
namespace {

struct NormParams {
  long long rows, xs, dys;  // xs, dys: distance of rows in elements
  int C, tpr;
  float eps;
};

constexpr int NORM_ROW_THREADS = 128;  // threads of a CTA whose rows lie within warps
constexpr int NORM_CTA = 512;          // of one whose rows span warps

// Sum over the `width` adjacent lanes (a power of two up to 32) that share a row.
__device__ __forceinline__ float lanes_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Barrier of the tpr threads (a multiple of 32) that share a row.
__device__ __forceinline__ void row_sync(int slot, int tpr) {
  asm volatile("bar.sync %0, %1;" ::"r"(slot + 1), "r"(tpr) : "memory");
}

// Valid elements among the vectors that the 32 lanes of a row's warp w hold.
template <int V, int NV> __device__ __forceinline__ float warp_count(int C, int tpr, int w) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int left = C / V - (j * tpr + w * 32);
    n += left <= 0 ? 0 : (left > 32 ? 32 : left);
  }
  return (float)(n * V);
}

// A thread's part of a row: NV vectors of V elements, tpr vectors apart, zeros beyond the row.
template <typename T, int V, int NV> struct RowPart {
  using P = Pack<T, V>;
  // the values of one vector, two to an instruction; the second half of a vector of one element is a zero
  // that no sum takes in
  static constexpr int H = (V + 1) / 2;
  typename P::Raw raw[NV];
  __device__ __forceinline__ void load(const T *row, int lane, int tpr, int C, bool live) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * tpr + lane) * V;
      raw[j] = P::zero();
      if (live && c < C) raw[j] = P::load(row + c);
    }
  }
  __device__ __forceinline__ void get(int j, float2 (&v)[H]) const { unpack(raw[j], v); }
  static __device__ __forceinline__ void unpack(const typename P::Raw &r, float2 (&v)[H]) {
    float f[V];
    P::unpack(r, f);
#pragma unroll
    for (int h = 0; h < H; ++h) v[h] = make_float2(f[2 * h], V > 1 ? f[(2 * h + 1) % V] : 0.f);
  }
  static __device__ __forceinline__ typename P::Raw pack(const float2 (&v)[H]) {
    float f[V];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      f[2 * h] = v[h].x;
      if (V > 1) f[(2 * h + 1) % V] = v[h].y;
    }
    return P::pack(f);
  }
  static __device__ __forceinline__ float total(float2 v) { return V > 1 ? v.x + v.y : v.x; }
};

// BLOCK: rows of tpr > 32 threads, blockDim / tpr of them at a time; otherwise 32 / tpr rows per warp.
template <typename T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? NORM_CTA : NORM_ROW_THREADS, BLOCK ? 2 : (V * NV > 24 ? 4 : 6))
norm_forward_kernel(const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ b, T *__restrict__ y,
                    float2 *stats, NormParams p) {
  using R = RowPart<T, V, NV>;
  using P = typename R::P;
  constexpr int H = R::H;
  __shared__ float2 red[2][NORM_CTA / 32];
  const int tpr = p.tpr, lane = threadIdx.x & (tpr - 1), slot = threadIdx.x / tpr, slots = blockDim.x / tpr;
  R next;
  const float inv = 1.f / (float)p.C;
  const int nw = tpr >> 5, wid = lane >> 5, other = BLOCK ? threadIdx.x & (nw - 1) : 0;
  // this warp's elements, and those of the warp whose moments this lane folds
  const float mine_n = BLOCK ? warp_count<V, NV>(p.C, tpr, wid) : 0.f;
  const float mine_inv = mine_n > 0.f ? 1.f / mine_n : 0.f;
  const float other_n = BLOCK ? warp_count<V, NV>(p.C, tpr, other) : 0.f;
  const long long step = (long long)gridDim.x * slots;
  int phase = 0;
  long long r = (long long)blockIdx.x * slots + slot;
  next.load(x + r * p.xs, lane, tpr, p.C, r < p.rows);
  // the rows of a warp go on together (shuffles); those of different warps need not
  for (long long r0 = BLOCK ? r : (long long)blockIdx.x * slots; r0 < p.rows; r0 += step, r += step) {
    const bool live = r < p.rows;
    float2 f[NV][H];
#pragma unroll
    for (int j = 0; j < NV; ++j) next.get(j, f[j]);
    next.load(x + (r + step) * p.xs, lane, tpr, p.C, r + step < p.rows);
    float2 sum2 = f2(0.f), sq2 = f2(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int h = 0; h < H; ++h) sum2 = add2(sum2, f[j][h]);
    const float sum = lanes_sum(R::total(sum2), BLOCK ? 32 : tpr);
    float mean = sum * (BLOCK ? mine_inv : inv);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if ((j * tpr + lane) * V < p.C) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float2 d = add2(f[j][h], f2(-mean));
          sq2 = fma2(d, d, sq2);
        }
      }
    float sq = lanes_sum(R::total(sq2), BLOCK ? 32 : tpr);
    if constexpr (BLOCK) {
      float2 *mine = red[phase] + slot * nw;
      if ((threadIdx.x & 31) == 0) mine[wid] = make_float2(mean, sq);
      row_sync(slot, tpr);
      const float2 o = mine[other];
      mean = lanes_sum(other_n * o.x, nw) * inv;
      const float d = o.x - mean;
      sq = lanes_sum(fmaf(other_n * d, d, o.y), nw);
      phase ^= 1;  // the other half: a fast warp may be a row ahead, never two
    }
    const float rstd = rsqrtf(sq * inv + p.eps);
    if (stats != nullptr && live && lane == 0) stats[r] = make_float2(mean, rstd);
    T *yr = y + r * p.C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * tpr + lane) * V;
      if (!live || c >= p.C) continue;
      float2 wv[H], bv[H];  // out of L1
#pragma unroll
      for (int h = 0; h < H; ++h) {
        wv[h] = f2(1.f);
        bv[h] = f2(0.f);
      }
      if (w) R::unpack(P::load(w + c), wv);
      if (b) R::unpack(P::load(b + c), bv);
#pragma unroll
      for (int h = 0; h < H; ++h) f[j][h] = fma2(mul2(add2(f[j][h], f2(-mean)), f2(rstd)), wv[h], bv[h]);
      P::store(yr + c, R::pack(f[j]));
    }
  }
}

// dx, and this CTA's part of dw and db: part[blockIdx.x][2][C].  Shared memory: [2][NV * tpr * V] floats.
template <typename T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? NORM_CTA : NORM_ROW_THREADS, BLOCK ? 1 : 4)
norm_backward_kernel(const T *__restrict__ x, const T *__restrict__ w, const float2 *__restrict__ stats,
                     const T *__restrict__ dy, T *__restrict__ dx, float *__restrict__ part, NormParams p) {
  using R = RowPart<T, V, NV>;
  using P = typename R::P;
  constexpr int H = R::H;
  __shared__ float2 red[2][NORM_CTA / 32];
  extern __shared__ float acc_s[];
  const int tpr = p.tpr, lane = threadIdx.x & (tpr - 1), slot = threadIdx.x / tpr, slots = blockDim.x / tpr;
  float2 dw[NV][H], db[NV][H];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int h = 0; h < H; ++h) dw[j][h] = db[j][h] = f2(0.f);
  R nx, ng, wr;
  if (w) wr.load(w, lane, tpr, p.C, true);
  const float inv = 1.f / (float)p.C;
  const int nw = tpr >> 5;
  const long long step = (long long)gridDim.x * slots;
  int phase = 0;
  long long r = (long long)blockIdx.x * slots + slot;
  nx.load(x + r * p.xs, lane, tpr, p.C, r < p.rows);
  ng.load(dy + r * p.dys, lane, tpr, p.C, r < p.rows);
  float2 ns = r < p.rows ? stats[r] : make_float2(0.f, 0.f);
  for (long long r0 = BLOCK ? r : (long long)blockIdx.x * slots; r0 < p.rows; r0 += step, r += step) {
    const bool live = r < p.rows, more = r + step < p.rows;
    const float2 st = ns;
    float2 xh[NV][H], g[NV][H];  // dy is zero beyond the row: what stands there counts nowhere
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      nx.get(j, xh[j]);
      ng.get(j, g[j]);
    }
    nx.load(x + (r + step) * p.xs, lane, tpr, p.C, more);
    ng.load(dy + (r + step) * p.dys, lane, tpr, p.C, more);
    ns = more ? stats[r + step] : make_float2(0.f, 0.f);
    float2 a1 = f2(0.f), a2 = f2(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float2 wv[H];
      if (w) wr.get(j, wv);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        xh[j][h] = mul2(add2(xh[j][h], f2(-st.x)), f2(st.y));
        dw[j][h] = fma2(g[j][h], xh[j][h], dw[j][h]);
        db[j][h] = add2(db[j][h], g[j][h]);
        if (w) g[j][h] = mul2(g[j][h], wv[h]);  // q from here on
        a1 = add2(a1, g[j][h]);
        a2 = fma2(g[j][h], xh[j][h], a2);
      }
    }
    float s1 = lanes_sum(R::total(a1), BLOCK ? 32 : tpr), s2 = lanes_sum(R::total(a2), BLOCK ? 32 : tpr);
    if constexpr (BLOCK) {
      float2 *mine = red[phase] + slot * nw;
      if ((threadIdx.x & 31) == 0) mine[lane >> 5] = make_float2(s1, s2);
      row_sync(slot, tpr);
      const float2 o = mine[threadIdx.x & (nw - 1)];
      s1 = lanes_sum(o.x, nw);
      s2 = lanes_sum(o.y, nw);
      phase ^= 1;
    }
    s1 *= inv * st.y;
    s2 *= inv * st.y;
    T *dr = dx + r * p.C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * tpr + lane) * V;
      if (!live || c >= p.C) continue;
      // rstd (q - mean(q) - xh mean(q xh))
#pragma unroll
      for (int h = 0; h < H; ++h) g[j][h] = fma2(g[j][h], f2(st.y), fma2(xh[j][h], f2(-s2), f2(-s1)));
      P::store(dr + c, R::pack(g[j]));
    }
  }
  if (part == nullptr) return;
  // rows of a warp by shuffles, then slot after slot (warp after warp) in order
  const int cols = NV * tpr * V, turns = BLOCK ? slots : (int)(blockDim.x >> 5);
  const int turn = BLOCK ? slot : (int)(threadIdx.x >> 5);
  auto each = [&](auto &&body) {  // body(value of dw, value of db, column)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i)
        body(i & 1 ? dw[j][i / 2].y : dw[j][i / 2].x, i & 1 ? db[j][i / 2].y : db[j][i / 2].x,
             (j * tpr + lane) * V + i);
  };
  if constexpr (!BLOCK)
    each([&](float &v, float &u, int) {
      for (int o = tpr; o < 32; o <<= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
        u += __shfl_xor_sync(0xffffffffu, u, o);
      }
    });
  for (int k = 0; k < turns; ++k) {
    if (turn == k && (BLOCK || (threadIdx.x & 31) < tpr))
      each([&](float &v, float &u, int c) {
        acc_s[c] = (k ? acc_s[c] : 0.f) + v;
        acc_s[cols + c] = (k ? acc_s[cols + c] : 0.f) + u;
      });
    __syncthreads();
  }
  float *mine = part + (long long)blockIdx.x * 2 * p.C;
  for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
    mine[c] = acc_s[c];
    mine[p.C + c] = acc_s[cols + c];
  }
}

// Rows too long for one CTA's registers: the row is read again for each step (from L2, mostly).
constexpr int WIDE_THREADS = 1024;

__device__ __forceinline__ float2 block_sum2(float a, float b, float2 *red) {
  a = warp_sum(a);
  b = warp_sum(b);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  a = b = 0.f;
  for (int i = 0; i < WIDE_THREADS / 32; ++i) {
    a += red[i].x;
    b += red[i].y;
  }
  return make_float2(a, b);
}

template <typename T>
__global__ void __launch_bounds__(WIDE_THREADS)
norm_forward_wide_kernel(const T *x, const T *w, const T *b, T *y, float2 *stats, NormParams p) {
  __shared__ float2 red[WIDE_THREADS / 32];
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T *xr = x + r * p.xs;
    float s = 0.f;
    for (int c = threadIdx.x; c < p.C; c += WIDE_THREADS) s += read(xr + c);
    const float mean = block_sum2(s, 0.f, red).x / (float)p.C;
    s = 0.f;
    for (int c = threadIdx.x; c < p.C; c += WIDE_THREADS) {
      const float d = read(xr + c) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = rsqrtf(block_sum2(s, 0.f, red).x / (float)p.C + p.eps);
    if (stats != nullptr && threadIdx.x == 0) stats[r] = make_float2(mean, rstd);
    for (int c = threadIdx.x; c < p.C; c += WIDE_THREADS) {
      const float v = (read(xr + c) - mean) * rstd;
      y[r * p.C + c] = Elem<T>::from_acc(fmaf(v, w ? read(w + c) : 1.f, b ? read(b + c) : 0.f));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(WIDE_THREADS)
norm_backward_wide_kernel(const T *x, const T *w, const float2 *stats, const T *dy, T *dx, float *part,
                          NormParams p) {
  __shared__ float2 red[WIDE_THREADS / 32];
  float *mine = part == nullptr ? nullptr : part + (long long)blockIdx.x * 2 * p.C;
  bool first = true;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T *xr = x + r * p.xs, *gr = dy + r * p.dys;
    const float2 st = stats[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < p.C; c += WIDE_THREADS) {
      const float q = read(gr + c) * (w ? read(w + c) : 1.f);
      s1 += q;
      s2 = fmaf(q, (read(xr + c) - st.x) * st.y, s2);
    }
    const float2 s = block_sum2(s1, s2, red);
    s1 = s.x / (float)p.C;
    s2 = s.y / (float)p.C;
    for (int c = threadIdx.x; c < p.C; c += WIDE_THREADS) {
      const float g = read(gr + c), xh = (read(xr + c) - st.x) * st.y;
      const float q = g * (w ? read(w + c) : 1.f);
      dx[r * p.C + c] = Elem<T>::from_acc(st.y * (q - s1 - xh * s2));
      if (mine) {  // a column belongs to one thread: no race
        mine[c] = (first ? 0.f : mine[c]) + g * xh;
        mine[p.C + c] = (first ? 0.f : mine[p.C + c]) + g;
      }
    }
    first = false;
  }
}

// ---- variant selection -------------------------------------------------------------------------

// Values of a row that a thread holds at most: rows within a warp, rows that span warps (whose CTAs have
// fewer registers per thread), and the backward pass, which keeps the sums of dw and db beside the row.
constexpr int NORM_MOST_WARP = 48, NORM_MOST = 16;

struct NormShape {
  int V, NV, tpr;  // tpr 0: the wide kernels
};

inline int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// The split of a row among threads that hold at most 16 values (8 in vectors of one element) with the
// fewest idle places; among equals the one with most values per thread (fewer steps in the row's sums, more
// bytes on their way).  `es`: bytes of an element, 0: vectors of one element only.
//
// With `most` = NORM_MOST_WARP also 3 and 6 vectors of 8, where they keep within a warp rows that would
// not fit one otherwise: no barriers.  Forward, 16 bits, against 3 vectors of 4: 200704 rows of 768, 113 us and
// 143; 131072 of 1536, 143 and 190; 200704 of 96, 22 and 25.  6 vectors are for rows that 3 do not hold (of 96:
// 24) and for more than a few per warp (8192 rows of 1536: 20 and 18).  4 vectors against 2 made no
// difference on rows of 64 to 1024 and are not in the choice.
//
// In 16 bits vectors of 4 are chosen by threes alone (a vector of 8 takes the place of two), and rows span warps
// only where threads hold the most that they may: nothing else is compiled (norm_spans_warps).
inline NormShape norm_shape(int C, int es, int most, long long rows) {
  static const NormShape choices[] = {{8, 1, 0}, {8, 2, 0}, {8, 3, 0}, {8, 6, 0}, {4, 1, 0}, {4, 2, 0},
                                      {4, 3, 0}, {4, 4, 0}, {1, 1, 0}, {1, 2, 0}, {1, 4, 0}, {1, 8, 0}};
  NormShape best{1, 0, 0};
  long long cost = 0;
  for (const NormShape &n : choices) {
    if (n.V * n.NV > most || (n.NV == 6 && rows < 16384) || (n.V == 4 && n.NV != 3 && es == 2)) continue;
    if (n.V != 1 ? (es == 0 || n.V * es > 16 || C % n.V != 0) : es != 0) continue;
    const int tpr = pow2_at_least(ceil_div(C / n.V, n.NV));
    if (tpr > (n.V * n.NV > NORM_MOST ? 32 : NORM_CTA) || (n.NV == 6 && tpr < 32)) continue;
    const long long places = (long long)tpr * n.NV * n.V;
    if (best.tpr == 0 || places < cost || (places == cost && n.V * n.NV > best.V * best.NV)) {
      best = NormShape{n.V, n.NV, tpr};
      cost = places;
    }
  }
  return best;
}

template <typename T, int V, int NV> constexpr bool norm_spans_warps() {
  return V * NV == (V == 1 ? 8 : NORM_MOST) || (V == 4 && NV == 3);
}

// CTAs: enough to fill every SM, each staying for many rows.
inline int norm_grid(long long rows, int slots, int per_sm) {
  const long long g = ceil_div_ll(rows, slots), most = 148ll * per_sm;
  return (int)(g < most ? g : most);
}
constexpr int NORM_PARTS = 148 * 4;  // most CTAs of the backward kernels, one part of the weight gradient each

template <typename T, int V, int NV>
void launch_forward(const T *x, const T *w, const T *b, T *y, float2 *stats, const NormParams &p, cudaStream_t st) {
  if constexpr (norm_spans_warps<T, V, NV>())
    if (p.tpr > 32) {
      norm_forward_kernel<T, V, NV, true>
          <<<norm_grid(p.rows, NORM_CTA / p.tpr, 2), NORM_CTA, 0, st>>>(x, w, b, y, stats, p);
      return;
    }
  if constexpr (V != 4 || sizeof(T) == 4)  // in 16 bits rows that vectors of 8 hold better
    norm_forward_kernel<T, V, NV, false>
        <<<norm_grid(p.rows, NORM_ROW_THREADS / p.tpr, 12), NORM_ROW_THREADS, 0, st>>>(x, w, b, y, stats, p);
}

template <typename T, int V, int NV>
int launch_backward(const T *x, const T *w, const float2 *stats, const T *dy, T *dx, float *part,
                    const NormParams &p, cudaStream_t st) {
  const size_t smem = part ? 2 * NV * p.tpr * V * sizeof(float) : 0;
  if constexpr (norm_spans_warps<T, V, NV>())
    if (p.tpr > 32) {
      const int grid = norm_grid(p.rows, NORM_CTA / p.tpr, 1);
      if (smem > 40 * 1024)
        (void)cudaFuncSetAttribute(norm_backward_kernel<T, V, NV, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   2 * NV * NORM_CTA * V * (int)sizeof(float));
      norm_backward_kernel<T, V, NV, true><<<grid, NORM_CTA, smem, st>>>(x, w, stats, dy, dx, part, p);
      return grid;
    }
  const int grid = norm_grid(p.rows, NORM_ROW_THREADS / p.tpr, 4);
  norm_backward_kernel<T, V, NV, false><<<grid, NORM_ROW_THREADS, smem, st>>>(x, w, stats, dy, dx, part, p);
  return grid;
}

// FN<T, V, NV>(...) for the shape `sh`
#define DWB_NORM_SWITCH(FN, ...)                            \
  switch (sh.V * 100 + sh.NV) {                             \
    case 101: FN<T, 1, 1>(__VA_ARGS__); break;              \
    case 102: FN<T, 1, 2>(__VA_ARGS__); break;              \
    case 104: FN<T, 1, 4>(__VA_ARGS__); break;              \
    case 108: FN<T, 1, 8>(__VA_ARGS__); break;              \
    default:                                                \
      if constexpr (sizeof(T) == 4) {                       \
        if (sh.NV == 1) FN<T, 4, 1>(__VA_ARGS__);           \
        else if (sh.NV == 2) FN<T, 4, 2>(__VA_ARGS__);      \
        else if (sh.NV == 3) FN<T, 4, 3>(__VA_ARGS__);      \
        else FN<T, 4, 4>(__VA_ARGS__);                      \
      } else {                                              \
        if (sh.V == 4) FN<T, 4, 3>(__VA_ARGS__);            \
        else if (sh.NV == 1) FN<T, 8, 1>(__VA_ARGS__);      \
        else FN<T, 8, 2>(__VA_ARGS__);                      \
      }                                                     \
  }

template <typename T>
void forward_t(const void *xv, const void *wv, const void *bv, void *yv, float *stats, NormParams p, cudaStream_t st) {
  const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv), *b = static_cast<const T *>(bv);
  T *y = static_cast<T *>(yv);
  float2 *s2 = reinterpret_cast<float2 *>(stats);
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.C % V == 0 && p.xs % V == 0 && aligned_to(x, 16) && aligned_to(y, 16) &&
                   (!w || aligned_to(w, 16)) && (!b || aligned_to(b, 16));
  const NormShape sh = norm_shape(p.C, vec ? (int)sizeof(T) : 0, NORM_MOST_WARP, p.rows);
  p.tpr = sh.tpr;
  if (sh.tpr == 0) {
    const int grid = (int)(p.rows < 148 * 2 ? p.rows : 148 * 2);
    norm_forward_wide_kernel<T><<<grid, WIDE_THREADS, 0, st>>>(x, w, b, y, s2, p);
    return;
  }
  if constexpr (sizeof(T) == 2)
    if (sh.V == 8 && sh.NV >= 3)
      return sh.NV == 3 ? launch_forward<T, 8, 3>(x, w, b, y, s2, p, st) : launch_forward<T, 8, 6>(x, w, b, y, s2, p, st);
  DWB_NORM_SWITCH(launch_forward, x, w, b, y, s2, p, st)
}

// Returns the parts of the weight gradient.
template <typename T>
int backward_t(const void *xv, const void *wv, const float *stats, const void *dyv, void *dxv, float *part,
               NormParams p, cudaStream_t st) {
  const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv), *dy = static_cast<const T *>(dyv);
  T *dx = static_cast<T *>(dxv);
  const float2 *s2 = reinterpret_cast<const float2 *>(stats);
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.C % V == 0 && p.xs % V == 0 && p.dys % V == 0 && aligned_to(x, 16) && aligned_to(dy, 16) &&
                   aligned_to(dx, 16) && (!w || aligned_to(w, 16));
  const NormShape sh = norm_shape(p.C, vec ? (int)sizeof(T) : 0, NORM_MOST, p.rows);
  p.tpr = sh.tpr;
  int parts = (int)(p.rows < 148 * 2 ? p.rows : 148 * 2);
  if (sh.tpr == 0) {
    norm_backward_wide_kernel<T><<<parts, WIDE_THREADS, 0, st>>>(x, w, s2, dy, dx, part, p);
    return parts;
  }
  DWB_NORM_SWITCH(parts = launch_backward, x, w, s2, dy, dx, part, p, st)
  return parts;
}

int check_norm(int dtype, long long rows, int C) {
  if (!seq_dtype_ok(dtype)) return DWCONV_B200_UNSUPPORTED_DTYPE;
  if (rows < 0 || C <= 0) return DWCONV_B200_BAD_ARGUMENT;
  if (C > (1 << 26)) return DWCONV_B200_TOO_LARGE;
  return DWCONV_B200_OK;
}

}  // namespace
}  // namespace dwb

using namespace dwb;

extern "C" {

int dwconv_b200_layer_norm(const void *x, long long x_stride, const void *w, const void *b, void *y,
                           float *stats, int dtype, long long rows, int C, float eps, void *stream) {
  int e = check_norm(dtype, rows, C);
  if (e) return e;
  if (x == nullptr || y == nullptr || !(eps >= 0.f)) return DWCONV_B200_BAD_ARGUMENT;
  const size_t es = elem_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(y, es) || (w && !aligned_to(w, es)) || (b && !aligned_to(b, es)) ||
      (stats && !aligned_to(stats, 8)))
    return DWCONV_B200_MISALIGNED;
  if (rows == 0) return DWCONV_B200_OK;
  const NormParams p{rows, x_stride, 0, C, 0, eps};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: forward_t<float>(x, w, b, y, stats, p, st); break;
    case DWCONV_B200_F16: forward_t<__half>(x, w, b, y, stats, p, st); break;
    default: forward_t<__nv_bfloat16>(x, w, b, y, stats, p, st); break;
  }
  return api_launch_status();
}

size_t dwconv_b200_layer_norm_workspace_bytes(int dtype, long long rows, int C) {
  if (check_norm(dtype, rows, C) != DWCONV_B200_OK) return 0;
  const size_t n = (size_t)(rows < NORM_PARTS ? rows : NORM_PARTS) * 2 * C * sizeof(float);
  return (n + 15) / 16 * 16 + 16;
}

int dwconv_b200_layer_norm_backward(const void *x, long long x_stride, const void *w, const float *stats,
                                    const void *dy, long long dy_stride, void *dx, void *dw, void *db,
                                    void *workspace, size_t workspace_bytes, int dtype, long long rows,
                                    int C, void *stream) {
  int e = check_norm(dtype, rows, C);
  if (e) return e;
  const bool params = dw != nullptr || db != nullptr;
  if (x == nullptr || stats == nullptr || dy == nullptr || dx == nullptr || (params && workspace == nullptr))
    return DWCONV_B200_BAD_ARGUMENT;
  const size_t es = elem_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(dy, es) || !aligned_to(dx, es) || (w && !aligned_to(w, es)) ||
      (dw && !aligned_to(dw, es)) || (db && !aligned_to(db, es)) || !aligned_to(stats, 8) ||
      (params && !aligned_to(workspace, 16)))
    return DWCONV_B200_MISALIGNED;
  if (params && workspace_bytes < dwconv_b200_layer_norm_workspace_bytes(dtype, rows, C))
    return DWCONV_B200_WORKSPACE_TOO_SMALL;
  const NormParams p{rows, x_stride, dy_stride, C, 0, 0.f};
  cudaStream_t st = (cudaStream_t)stream;
  float *part = params ? static_cast<float *>(workspace) : nullptr;
  int parts = 0;
  if (rows > 0) {
    switch (dtype) {
      case DWCONV_B200_F32: parts = backward_t<float>(x, w, stats, dy, dx, part, p, st); break;
      case DWCONV_B200_F16: parts = backward_t<__half>(x, w, stats, dy, dx, part, p, st); break;
      default: parts = backward_t<__nv_bfloat16>(x, w, stats, dy, dx, part, p, st); break;
    }
    e = api_launch_status();
    if (e) return e;
  }
  if (params) launch_column_sum(part, parts, 2 * C, ColumnSumOut{dw, db, dtype, C, 1, nullptr}, st);
  return api_launch_status();
}

}  // extern "C"
