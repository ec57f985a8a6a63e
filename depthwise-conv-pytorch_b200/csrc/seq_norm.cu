// Layer norm over the channels of a row, forward and backward (declarations: include/dwconv_b200.h).
//
//   y = (x - m) s w + b,  m = mean, s = 1 / sqrt(mean (x - m)^2 + eps)
//   with xh = (x - m) s and q = dy w:   dx = s (q - mean(q) - xh mean(q xh)),
//   dw = sum over rows of dy xh,  db = sum over rows of dy.
//
// Both directions read each row once: `tpr` threads own a row (a power of two, up to a whole CTA) and
// keep its values in registers, NV vectors of V elements per thread.  The variance is the sum of
// squares around the mean (warps' sums are merged by the parallel-variance formula, so that one
// exchange through shared memory gives both moments), never a difference of large sums.
#include "seq_common.cuh"

namespace dwb {
namespace {

struct NormParams {
  long long rows, xs, dys;  // xs, dys: distance of rows in elements
  int C, tpr;
  float eps;
};

constexpr int NORM_WARPS = 32;
constexpr int NORM_ROW_THREADS = 128;  // threads of a CTA that holds several rows

// Most threads that share a row whose threads hold `per` values each: what the registers of one SM
// allow (forward: the values; backward: x, dy, w and the two running sums).
__host__ __device__ constexpr int norm_max_tpr(int per, bool backward) {
  return backward ? (per <= 4 ? 1024 : per <= 16 ? 512 : 256) : (per <= 16 ? 1024 : 512);
}

// Sum over the `width` adjacent lanes (a power of two up to 32) that share a row.
__device__ __forceinline__ float lanes_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Valid elements among the vectors that the 32 lanes of warp w hold.
template <int V, int NV> __device__ __forceinline__ float warp_count(int C, int tpr, int w) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int left = C / V - (j * tpr + w * 32);
    n += left <= 0 ? 0 : (left > 32 ? 32 : left);
  }
  return (float)(n * V);
}

// BLOCK: a CTA of tpr > 32 threads per row; otherwise 32 / tpr rows per warp.
template <typename T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? norm_max_tpr(V *NV, false) : NORM_ROW_THREADS)
norm_forward_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                    const T *__restrict__ b, T *__restrict__ y, float2 *stats, NormParams p) {
  using P = Pack<T, V>;
  __shared__ float2 red[2][BLOCK ? NORM_WARPS : 1];
  const int tid = threadIdx.x, lane = tid & (p.tpr - 1);
  const int slots = BLOCK ? 1 : blockDim.x / p.tpr;
  const int slot = BLOCK ? 0 : tid / p.tpr;
  int phase = 0;
  for (long long r0 = (long long)blockIdx.x * slots; r0 < p.rows; r0 += (long long)gridDim.x * slots) {
    const long long r = r0 + slot;
    const bool live = r < p.rows;
    float f[NV][V];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * p.tpr + lane) * V;
      typename P::Raw raw = P::zero();
      if (live && c < p.C) raw = P::load(x + r * p.xs + c);
      P::unpack(raw, f[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) sum += f[j][i];
    }
    float mean, rstd;
    if constexpr (!BLOCK) {
      mean = lanes_sum(sum, p.tpr) / (float)p.C;
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((j * p.tpr + lane) * V < p.C) {
#pragma unroll
          for (int i = 0; i < V; ++i) sq += (f[j][i] - mean) * (f[j][i] - mean);
        }
      rstd = rsqrtf(lanes_sum(sq, p.tpr) / (float)p.C + p.eps);
    } else {
      const int wid = tid >> 5, nw = p.tpr >> 5;
      const float n = warp_count<V, NV>(p.C, p.tpr, wid);
      const float wm = n > 0.f ? lanes_sum(sum, 32) / n : 0.f;
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((j * p.tpr + lane) * V < p.C) {
#pragma unroll
          for (int i = 0; i < V; ++i) sq += (f[j][i] - wm) * (f[j][i] - wm);
        }
      sq = lanes_sum(sq, 32);
      if ((tid & 31) == 0) red[phase][wid] = make_float2(wm, sq);
      __syncthreads();
      float m = 0.f, m2 = 0.f;
      for (int i = 0; i < nw; ++i) m += warp_count<V, NV>(p.C, p.tpr, i) * red[phase][i].x;
      m /= (float)p.C;
      for (int i = 0; i < nw; ++i) {
        const float d = red[phase][i].x - m;
        m2 += red[phase][i].y + warp_count<V, NV>(p.C, p.tpr, i) * d * d;
      }
      mean = m;
      rstd = rsqrtf(m2 / (float)p.C + p.eps);
      phase ^= 1;  // the other half: a fast warp may be a row ahead, never two
    }
    if (stats != nullptr && live && lane == 0) stats[r] = make_float2(mean, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * p.tpr + lane) * V;
      if (!live || c >= p.C) continue;
      float wv[V], bv[V];
      if (w) P::unpack(P::load(w + c), wv);
      if (b) P::unpack(P::load(b + c), bv);
#pragma unroll
      for (int i = 0; i < V; ++i)
        f[j][i] = fmaf((f[j][i] - mean) * rstd, w ? wv[i] : 1.f, b ? bv[i] : 0.f);
      P::store(y + r * p.C + c, P::pack(f[j]));
    }
  }
}

// dx, and this CTA's part of dw and db: part[blockIdx.x][2][C].
template <typename T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? norm_max_tpr(V *NV, true) : NORM_ROW_THREADS)
norm_backward_kernel(const T *__restrict__ x, const T *__restrict__ w,
                                     const float2 *__restrict__ stats, const T *__restrict__ dy,
                                     T *__restrict__ dx, float *__restrict__ part, NormParams p) {
  using P = Pack<T, V>;
  __shared__ float2 red[2][BLOCK ? NORM_WARPS : 1];
  extern __shared__ float acc_s[];  // !BLOCK: [2][NV * tpr * V]
  const int tid = threadIdx.x, lane = tid & (p.tpr - 1);
  const int slots = BLOCK ? 1 : blockDim.x / p.tpr;
  const int slot = BLOCK ? 0 : tid / p.tpr;
  float dw[NV][V], db[NV][V], wv[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * p.tpr + lane) * V;
    typename P::Raw raw = P::zero();
    if (w && c < p.C) raw = P::load(w + c);
    P::unpack(raw, wv[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[j][i] = db[j][i] = 0.f;
      if (!w) wv[j][i] = 1.f;
    }
  }
  const float inv = 1.f / (float)p.C;
  int phase = 0;
  for (long long r0 = (long long)blockIdx.x * slots; r0 < p.rows; r0 += (long long)gridDim.x * slots) {
    const long long r = r0 + slot;
    const bool live = r < p.rows;
    const float2 st = live ? stats[r] : make_float2(0.f, 0.f);
    float xh[NV][V], g[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * p.tpr + lane) * V;
      typename P::Raw rx = P::zero(), rg = P::zero();
      const bool on = live && c < p.C;
      if (on) {
        rx = P::load(x + r * p.xs + c);
        rg = P::load(dy + r * p.dys + c);
      }
      P::unpack(rx, xh[j]);
      P::unpack(rg, g[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[j][i] = on ? (xh[j][i] - st.x) * st.y : 0.f;
        const float q = g[j][i] * wv[j][i];
        s1 += q;
        s2 = fmaf(q, xh[j][i], s2);
        dw[j][i] = fmaf(g[j][i], xh[j][i], dw[j][i]);
        db[j][i] += g[j][i];
      }
    }
    if constexpr (!BLOCK) {
      s1 = lanes_sum(s1, p.tpr);
      s2 = lanes_sum(s2, p.tpr);
    } else {
      s1 = lanes_sum(s1, 32);
      s2 = lanes_sum(s2, 32);
      if ((tid & 31) == 0) red[phase][tid >> 5] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.f;
      for (int i = 0; i < (p.tpr >> 5); ++i) {
        s1 += red[phase][i].x;
        s2 += red[phase][i].y;
      }
      phase ^= 1;
    }
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * p.tpr + lane) * V;
      if (!live || c >= p.C) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = st.y * (g[j][i] * wv[j][i] - s1 - xh[j][i] * s2);
      P::store(dx + r * p.C + c, P::pack(o));
    }
  }
  if (part == nullptr) return;
  float *mine = part + (long long)blockIdx.x * 2 * p.C;
  if constexpr (BLOCK) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * p.tpr + lane) * V;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < p.C) {
          mine[c + i] = dw[j][i];
          mine[p.C + c + i] = db[j][i];
        }
    }
  } else {
    // rows of a warp by shuffles, then warp after warp in order
    const int cols = NV * p.tpr * V;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i)
        for (int o = p.tpr; o < 32; o <<= 1) {
          dw[j][i] += __shfl_xor_sync(0xffffffffu, dw[j][i], o);
          db[j][i] += __shfl_xor_sync(0xffffffffu, db[j][i], o);
        }
    for (int k = 0; k < (int)(blockDim.x >> 5); ++k) {
      if ((tid >> 5) == k && (tid & 31) < p.tpr) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int c = (j * p.tpr + lane) * V + i;
            acc_s[c] = (k ? acc_s[c] : 0.f) + dw[j][i];
            acc_s[cols + c] = (k ? acc_s[cols + c] : 0.f) + db[j][i];
          }
      }
      __syncthreads();
    }
    for (int c = tid; c < p.C; c += blockDim.x) {
      mine[c] = acc_s[c];
      mine[p.C + c] = acc_s[cols + c];
    }
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

struct NormShape {
  int V, NV, tpr;  // tpr 0: the wide kernels
};

inline int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// The split of a row with the fewest idle places; among equals the one with most values per thread
// (fewer steps in the row's sums).
inline NormShape norm_shape(int C, int V, bool backward) {
  static const int nv16[] = {1, 2, 3, 0}, nv8[] = {1, 2, 3, 4, 0}, nv1[] = {1, 2, 4, 8, 16, 0};
  const int *nv = V == 8 ? nv16 : V == 4 ? nv8 : nv1;
  NormShape best{V, 0, 0};
  long long cost = 0;
  for (; *nv; ++nv) {
    const int tpr = pow2_at_least(ceil_div(C / V, *nv));
    if (tpr > norm_max_tpr(V * *nv, backward)) continue;
    if (best.tpr == 0 || (long long)tpr * *nv <= cost) {
      best = NormShape{V, *nv, tpr};
      cost = (long long)tpr * *nv;
    }
  }
  return best;
}

inline int norm_forward_grid(long long rows, int slots) {
  const long long g = ceil_div_ll(rows, slots), cap = 148ll * 64;
  return (int)(g < cap ? g : cap);
}
// CTAs of the backward kernels, one part of the weight gradient each.
inline int norm_backward_parts(long long rows) { return (int)(rows < 148 * 4 ? rows : 148 * 4); }

template <typename T, int V, int NV>
void launch_forward(const T *x, const T *w, const T *b, T *y, float2 *stats, const NormParams &p, cudaStream_t st) {
  if (p.tpr > 32)
    norm_forward_kernel<T, V, NV, true><<<norm_forward_grid(p.rows, 1), p.tpr, 0, st>>>(x, w, b, y, stats, p);
  else
    norm_forward_kernel<T, V, NV, false>
        <<<norm_forward_grid(p.rows, NORM_ROW_THREADS / p.tpr), NORM_ROW_THREADS, 0, st>>>(x, w, b, y, stats, p);
}

template <typename T, int V, int NV>
void launch_backward(const T *x, const T *w, const float2 *stats, const T *dy, T *dx, float *part, int parts,
                     const NormParams &p, cudaStream_t st) {
  if (p.tpr > 32)
    norm_backward_kernel<T, V, NV, true><<<parts, p.tpr, 0, st>>>(x, w, stats, dy, dx, part, p);
  else
    norm_backward_kernel<T, V, NV, false><<<parts, NORM_ROW_THREADS, 2 * NV * p.tpr * V * sizeof(float), st>>>(
        x, w, stats, dy, dx, part, p);
}

#define DWB_NORM_SWITCH(FN, ...)                                        \
  switch (sh.V * 100 + sh.NV) {                                         \
    case 101: FN<T, 1, 1>(__VA_ARGS__); break;                          \
    case 102: FN<T, 1, 2>(__VA_ARGS__); break;                          \
    case 104: FN<T, 1, 4>(__VA_ARGS__); break;                          \
    case 108: FN<T, 1, 8>(__VA_ARGS__); break;                          \
    case 116: FN<T, 1, 16>(__VA_ARGS__); break;                         \
    default: FN##_vec<T, 16 / (int)sizeof(T)>(__VA_ARGS__, sh.NV); break; \
  }


template <typename T, int V>
void launch_forward_vec(const T *x, const T *w, const T *b, T *y, float2 *stats, const NormParams &p,
                        cudaStream_t st, int nv) {
  switch (nv) {
    case 1: launch_forward<T, V, 1>(x, w, b, y, stats, p, st); break;
    case 2: launch_forward<T, V, 2>(x, w, b, y, stats, p, st); break;
    case 3: launch_forward<T, V, 3>(x, w, b, y, stats, p, st); break;
    default:
      if constexpr (V == 4) launch_forward<T, V, 4>(x, w, b, y, stats, p, st);
  }
}
template <typename T, int V>
void launch_backward_vec(const T *x, const T *w, const float2 *stats, const T *dy, T *dx, float *part, int parts,
                         const NormParams &p, cudaStream_t st, int nv) {
  switch (nv) {
    case 1: launch_backward<T, V, 1>(x, w, stats, dy, dx, part, parts, p, st); break;
    case 2: launch_backward<T, V, 2>(x, w, stats, dy, dx, part, parts, p, st); break;
    case 3: launch_backward<T, V, 3>(x, w, stats, dy, dx, part, parts, p, st); break;
    default:
      if constexpr (V == 4) launch_backward<T, V, 4>(x, w, stats, dy, dx, part, parts, p, st);
  }
}

template <typename T>
void forward_t(const void *xv, const void *wv, const void *bv, void *yv, float *stats, NormParams p, cudaStream_t st) {
  const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv), *b = static_cast<const T *>(bv);
  T *y = static_cast<T *>(yv);
  float2 *s2 = reinterpret_cast<float2 *>(stats);
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.C % V == 0 && p.xs % V == 0 && aligned_to(x, 16) && aligned_to(y, 16) &&
                   (!w || aligned_to(w, 16)) && (!b || aligned_to(b, 16));
  const NormShape sh = norm_shape(p.C, vec ? V : 1, false);
  p.tpr = sh.tpr;
  if (sh.tpr == 0) {
    const int grid = (int)(p.rows < 148 * 2 ? p.rows : 148 * 2);
    norm_forward_wide_kernel<T><<<grid, WIDE_THREADS, 0, st>>>(x, w, b, y, s2, p);
    return;
  }
  DWB_NORM_SWITCH(launch_forward, x, w, b, y, s2, p, st)
}

template <typename T>
void backward_t(const void *xv, const void *wv, const float *stats, const void *dyv, void *dxv, float *part,
                int parts, NormParams p, cudaStream_t st) {
  const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv), *dy = static_cast<const T *>(dyv);
  T *dx = static_cast<T *>(dxv);
  const float2 *s2 = reinterpret_cast<const float2 *>(stats);
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.C % V == 0 && p.xs % V == 0 && p.dys % V == 0 && aligned_to(x, 16) && aligned_to(dy, 16) &&
                   aligned_to(dx, 16) && (!w || aligned_to(w, 16));
  const NormShape sh = norm_shape(p.C, vec ? V : 1, true);
  p.tpr = sh.tpr;
  if (sh.tpr == 0) {
    norm_backward_wide_kernel<T><<<parts, WIDE_THREADS, 0, st>>>(x, w, s2, dy, dx, part, p);
    return;
  }
  DWB_NORM_SWITCH(launch_backward, x, w, s2, dy, dx, part, parts, p, st)
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
  const size_t n = (size_t)norm_backward_parts(rows) * 2 * C * sizeof(float);
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
  const int parts = norm_backward_parts(rows);
  if (rows > 0) {
    switch (dtype) {
      case DWCONV_B200_F32: backward_t<float>(x, w, stats, dy, dx, part, parts, p, st); break;
      case DWCONV_B200_F16: backward_t<__half>(x, w, stats, dy, dx, part, parts, p, st); break;
      default: backward_t<__nv_bfloat16>(x, w, stats, dy, dx, part, parts, p, st); break;
    }
    e = api_launch_status();
    if (e) return e;
  }
  if (params) launch_column_sum(part, parts, 2 * C, ColumnSumOut{dw, db, dtype, C, 1, nullptr}, st);
  return api_launch_status();
}

}  // extern "C"
