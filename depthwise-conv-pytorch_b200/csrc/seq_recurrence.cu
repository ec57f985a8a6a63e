// Gated linear recurrence over [B, T, C] sequences: a scan along T with its gates computed on the
// way, the backward pass, and the one-row step (declarations: include/dwconv_b200.h).
//
//   r = sigmoid(u), i = sigmoid(v), z = scale softplus(decay) r
//   d = 1 - exp(-z),  a = 1 - d,  beta = sqrt(1 - a^2) = sqrt(d (2 - d))
//   h[t] = a h[t-1] + beta i x,   y = h
// and with g[t] = dy[t] + a[t+1] g[t+1]:
//   dx = g beta i,  dv = dx x (1 - i),  dz = g (a^2 / beta i x - a h[t-1]),  du = dz z (1 - r),
//   ddecay = scale sigmoid(decay) sum_t dz r,  dinitial = a[0] g[0].
// d, not a, is what is computed: for the long memories such models use z is small, and 1 - exp(-z)
// by its power series keeps both 1 - a and beta to a few units in the last place.
//
// Bound by memory: forward x, u, v in and y out; backward x, u, v, dy in and dx, du, dv out.
//
// Layout.  A lane owns two channels, a warp 64 channels of L consecutive rows, a CTA of W warps a tile
// of W * L rows.  A warp reduces its rows to one pair (P, H): the state that leaves them is
// P h + H.  Pairs meet in shared memory, every warp folds those in front of it onto the state that
// enters the tile, and walks its rows once more from registers.  Tiles follow one another along T.
// Where there are too few (channel block, batch) pairs to fill the device, a cluster of CTAs takes
// neighbouring tiles together and passes its tiles' pairs through distributed shared memory: one
// cluster barrier per CTAs * W * L rows, no pass over the data for it, and the same order of
// operations on every run.
//
// The forward pass keeps the fp32 state that enters each tile (1 / (W L) of the rows); the backward
// pass starts from it, so it reads y nowhere and its h[t-1] have not been rounded to the data's type.
#include <mutex>

#include "seq_common.cuh"

namespace dwb {
namespace {

constexpr int REC_L = 8, REC_W = 8, REC_TILE = REC_L * REC_W, REC_GROUP = 64;
constexpr int REC_THREADS = REC_W * 32;
constexpr int REC_MAX_CLUSTER = 8;
// Largest z for which the power series is used alone: its first omitted term, z^6 / 5040 relative, is
// 5e-8 there.
constexpr float REC_SERIES = 0.25f;

// ---- arithmetic on channel pairs ---------------------------------------------------------------

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }

__device__ __forceinline__ float ex2f(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcpf(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rsqf(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float LOG2E = 1.4426950408889634f;

// 1 / (1 + 2^(-v log2 e)); an overflowing exponential gives 0.
__device__ __forceinline__ float2 sigmoid2(float2 v) {
  const float2 e = mul2(v, f2(-LOG2E));
  const float2 s = add2(make_float2(ex2f(e.x), ex2f(e.y)), f2(1.f));
  return make_float2(rcpf(s.x), rcpf(s.y));
}

// 1 - exp(-z), z >= 0.  `series`: every z of this warp is at most REC_SERIES.
__device__ __forceinline__ float2 decay2(float2 z, bool series) {
  float2 p = fma2(z, f2(-1.f / 720.f), f2(1.f / 120.f));
  p = fma2(p, neg2(z), f2(1.f / 24.f));
  p = fma2(p, neg2(z), f2(1.f / 6.f));
  p = fma2(p, neg2(z), f2(0.5f));
  p = fma2(p, neg2(z), f2(1.f));
  float2 d = mul2(z, p);
  if (!series) {
    const float2 e = mul2(z, f2(-LOG2E));
    if (!(z.x <= REC_SERIES)) d.x = 1.f - ex2f(e.x);
    if (!(z.y <= REC_SERIES)) d.y = 1.f - ex2f(e.y);
  }
  return d;
}

// a = exp(-z) from d = 1 - exp(-z): their difference from 1 where d is small, the exponential itself
// where a is, so that each is good to a few units in its own last place.
__device__ __forceinline__ float2 keep2(float2 z, float2 d, bool series) {
  float2 a = add2(f2(1.f), neg2(d));
  if (!series) {
    const float2 e = mul2(z, f2(-LOG2E));
    if (!(z.x <= REC_SERIES)) a.x = ex2f(e.x);
    if (!(z.y <= REC_SERIES)) a.y = ex2f(e.y);
  }
  return a;
}

// d (2 - d) = 1 - a^2, kept off zero so that its reciprocal root stays finite (z = 0: closed gate).
__device__ __forceinline__ float2 beta_square2(float2 d) {
  const float2 q = fma2(neg2(d), d, add2(d, d));
  float2 r;  // a NaN stays one
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r.x) : "f"(q.x), "f"(1e-37f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r.y) : "f"(q.y), "f"(1e-37f));
  return r;
}

struct Gates {
  float2 r, i, d;
};
__device__ __forceinline__ Gates gates(float2 u, float2 v, float2 kz, bool series) {
  Gates g;
  g.r = sigmoid2(u);
  g.i = sigmoid2(v);
  g.d = decay2(mul2(kz, g.r), series);
  return g;
}

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }

// ---- channel pairs of a lane -------------------------------------------------------------------

// VEC: channels c, c + 1, one load.  Otherwise (odd C, odd strides) channels c and c + 32, one each.
template <typename T, bool VEC> struct Pair;
template <typename T> struct Pair<T, true> {
  using P = Pack<T, 2>;
  using Raw = typename P::Raw;
  static __device__ __forceinline__ int channel(int g, int lane) { return g * REC_GROUP + 2 * lane; }
  static __device__ __forceinline__ Raw zero() { return P::zero(); }
  static __device__ __forceinline__ Raw load(const T *p, bool on0, bool) {
    return on0 ? P::load(p) : P::zero();
  }
  static __device__ __forceinline__ float2 get(const Raw &r) {
    float f[2];
    P::unpack(r, f);
    return make_float2(f[0], f[1]);
  }
  static __device__ __forceinline__ void store(T *p, float2 v, bool on0, bool) {
    const float f[2] = {v.x, v.y};
    if (on0) P::store(p, P::pack(f));
  }
};
template <typename T> struct Pair<T, false> {
  struct Raw { T a, b; };
  static __device__ __forceinline__ int channel(int g, int lane) { return g * REC_GROUP + lane; }
  static __device__ __forceinline__ Raw zero() { return Raw{Elem<T>::from_acc(0.f), Elem<T>::from_acc(0.f)}; }
  static __device__ __forceinline__ Raw load(const T *p, bool on0, bool on1) {
    Raw r = zero();
    if (on0) r.a = p[0];
    if (on1) r.b = p[32];
    return r;
  }
  static __device__ __forceinline__ float2 get(const Raw &r) {
    return make_float2(Elem<T>::to_acc(r.a), Elem<T>::to_acc(r.b));
  }
  static __device__ __forceinline__ void store(T *p, float2 v, bool on0, bool on1) {
    if (on0) p[0] = Elem<T>::from_acc(v.x);
    if (on1) p[32] = Elem<T>::from_acc(v.y);
  }
};

// ---- rows of a warp ----------------------------------------------------------------------------

// Which of a warp's L rows begin a sequence, end one, or belong to none (bit j: row t0 + j).
struct RowMasks {
  unsigned start, end, none;
};

struct RowWalk {
  SeqSpan sp;
  __device__ __forceinline__ void init(const SeqList &q, int b) {
    sp = q.offsets ? SeqSpan{-1, 0, 0} : SeqSpan{b, 0, q.T};
  }
  template <int L> __device__ __forceinline__ RowMasks masks(const SeqList &q, int t0) {
    RowMasks m{0u, 0u, 0u};
    if (q.offsets == nullptr || (sp.seq >= 0 && t0 >= sp.begin && t0 + L <= sp.next)) {
      if (t0 == sp.begin) m.start = 1u;
      const int last = sp.next - 1 - t0;
      if (last >= 0 && last < L) m.end = 1u << last;
      const int rows = q.T - t0;
      if (rows < L) m.none = rows <= 0 ? (1u << L) - 1u : ((1u << L) - 1u) & ~((1u << rows) - 1u);
      return m;
    }
    for (int j = 0; j < L; ++j) {
      const int t = t0 + j;
      if (t >= q.T) {
        m.none |= 1u << j;
        continue;
      }
      if (j == 0 || t == sp.next) sp = seq_locate(q, t);
      if (sp.seq < 0) {
        m.none |= 1u << j;
      } else {
        if (t == sp.begin) m.start |= 1u << j;
        if (t + 1 == sp.next) m.end |= 1u << j;
      }
    }
    return m;
  }
};

__device__ __forceinline__ int seq_index(const SeqList &q, int b, int t) {
  return q.offsets ? seq_locate(q, t).seq : b;
}

__device__ __forceinline__ float2 load_state(const float *s, long long j, int C, int c, int c1, bool on0, bool on1) {
  return make_float2(on0 ? s[j * C + c] : 0.f, on1 ? s[j * C + c1] : 0.f);
}
__device__ __forceinline__ void store_state(float *s, long long j, int C, int c, int c1, bool on0, bool on1, float2 v) {
  if (on0) s[j * C + c] = v.x;
  if (on1) s[j * C + c1] = v.y;
}

// A pair whose rows begin a sequence takes nothing from in front of it, whatever stands there (an
// infinity times zero would not be zero): its P is -1, which no product of decays is, and stays -1
// whatever it is multiplied by (a NaN would take the sign away).
__device__ __forceinline__ bool cut(float2 P) { return __float_as_int(P.x) < 0; }
__device__ __forceinline__ float2 join(float2 P, float2 Q) { return cut(P) || cut(Q) ? f2(-1.f) : mul2(P, Q); }
__device__ __forceinline__ float2 apply(float2 P, float2 H, float2 h) { return cut(P) ? H : fma2(P, h, H); }

// ---- thread-block clusters ---------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_peer(const void *mine, int rank, float4 v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(mine)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

struct RecParams {
  SeqList q;
  int B, groups, cs;  // cs: CTAs of a cluster
  float scale;
};

// Sequences without a row: what enters leaves.
__device__ __forceinline__ void empty_states(const RecParams &p, int b, int warp, const float *from, float *to, int c,
                                             int c1, bool on0, bool on1) {
  if (p.q.offsets == nullptr) {
    if (p.q.T == 0 && warp == 0)
      store_state(to, b, p.q.C, c, c1, on0, on1, from ? load_state(from, b, p.q.C, c, c1, on0, on1) : f2(0.f));
    return;
  }
  for (int j = warp; j < p.q.S; j += REC_W)
    if (seq_bound(p.q, j) >= seq_bound(p.q, j + 1))
      store_state(to, j, p.q.C, c, c1, on0, on1, from ? load_state(from, j, p.q.C, c, c1, on0, on1) : f2(0.f));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(REC_THREADS)
recurrence_forward_kernel(SeqIn<T> x, SeqIn<T> u, SeqIn<T> v, const float *__restrict__ decay,
                          const float *__restrict__ initial, T *__restrict__ y, float *__restrict__ fin,
                          float *__restrict__ ckpt, RecParams p) {
  using Q = Pair<T, VEC>;
  constexpr int L = REC_L, W = REC_W;
  __shared__ float4 agg[2][W][32];
  __shared__ float4 far[2][REC_MAX_CLUSTER][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = (int)(blockIdx.x % p.cs);
  const long long pair = blockIdx.x / p.cs;
  const int grp = (int)(pair % p.groups), b = (int)(pair / p.groups);
  const int C = p.q.C, c = Q::channel(grp, lane), c1 = VEC ? c + 1 : c + 32;
  const bool on0 = c < C, on1 = c1 < C;
  if (p.cs > 1) {  // a peer's shared memory may be written once it runs
    cluster_arrive();
    cluster_wait();
  }
  if (fin != nullptr && rank == 0) empty_states(p, b, warp, initial, fin, c, c1, on0, on1);
  const float2 kz = make_float2(on0 ? p.scale * softplus(decay[c]) : 0.f,
                                on1 ? p.scale * softplus(decay[c1]) : 0.f);
  const bool series = __all_sync(0xffffffffu, kz.x <= REC_SERIES && kz.y <= REC_SERIES);
  const int tiles = ceil_div(p.q.T, REC_TILE), steps = ceil_div(tiles, p.cs);
  RowWalk walk;
  walk.init(p.q, b);
  float2 carry = f2(0.f);
  for (int it = 0; it < steps; ++it) {
    const int tile = it * p.cs + rank, t0 = tile * REC_TILE + warp * L, half = it & 1;
    const RowMasks m = walk.masks<L>(p.q, t0);
    typename Q::Raw rx[L], ru[L], rv[L];
    {
      const T *px = x.row(b, t0) + c, *pu = u.row(b, t0) + c, *pv = v.row(b, t0) + c;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const bool in = !(m.none >> j & 1u);
        rx[j] = Q::load(px + j * x.rs, in && on0, in && on1);
        ru[j] = Q::load(pu + j * u.rs, in && on0, in && on1);
        rv[j] = Q::load(pv + j * v.rs, in && on0, in && on1);
      }
    }
    float2 a[L], bb[L], P = f2(1.f), H = f2(0.f);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const Gates g = gates(Q::get(ru[j]), Q::get(rv[j]), kz, series);
      const float2 q = beta_square2(g.d);
      a[j] = keep2(mul2(kz, g.r), g.d, series);
      bb[j] = mul2(mul2(q, make_float2(rsqf(q.x), rsqf(q.y))), mul2(g.i, Q::get(rx[j])));
    }
    if ((m.start | m.none) == 0u) {
#pragma unroll
      for (int j = 0; j < L; ++j) {
        P = mul2(P, a[j]);
        H = fma2(a[j], H, bb[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < L; ++j) {
        if (m.none >> j & 1u) {
          a[j] = bb[j] = f2(0.f);
          P = f2(-1.f);
          H = f2(0.f);
        } else if (m.start >> j & 1u) {
          if (initial != nullptr)
            bb[j] = fma2(a[j], load_state(initial, seq_index(p.q, b, t0 + j), C, c, c1, on0, on1), bb[j]);
          P = f2(-1.f);
          H = bb[j];
        } else {
          P = join(P, a[j]);
          H = fma2(a[j], H, bb[j]);
        }
      }
    }
    agg[half][warp][lane] = make_float4(P.x, P.y, H.x, H.y);
    __syncthreads();
    float2 h = carry;
    if (p.cs > 1) {
      // the CTA's pair, folded by as many warps as it has peers, one peer each
      if (warp < p.cs) {
        float2 TP = f2(1.f), TH = f2(0.f);
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float4 e = agg[half][k][lane];
          const float2 P2 = make_float2(e.x, e.y), H2 = make_float2(e.z, e.w);
          TH = apply(P2, H2, TH);
          TP = join(TP, P2);
        }
        store_peer(&far[half][rank][lane], warp, make_float4(TP.x, TP.y, TH.x, TH.y));
      }
      cluster_arrive();
      cluster_wait();
      for (int k = 0; k < p.cs; ++k) {
        if (k == rank) h = carry;
        const float4 e = far[half][k][lane];
        carry = apply(make_float2(e.x, e.y), make_float2(e.z, e.w), carry);
      }
    }
    if (ckpt != nullptr && warp == 0 && tile < tiles)
      store_state(ckpt, (long long)b * tiles + tile, C, c, c1, on0, on1, h);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if (p.cs > 1 && k == warp) break;
      const float4 e = agg[half][k][lane];
      if (k == warp) carry = h;  // cs 1: the state of this warp, while h runs on to the tile's end
      h = apply(make_float2(e.x, e.y), make_float2(e.z, e.w), h);
    }
    if (p.cs == 1) {
      const float2 next = h;
      h = carry;
      carry = next;
    }
    T *py = y + ((long long)b * p.q.T + t0) * C + c;
#pragma unroll
    for (int j = 0; j < L; ++j) {
      h = ((m.start | m.none) >> j & 1u) ? bb[j] : fma2(a[j], h, bb[j]);
      const bool in = t0 + j < p.q.T;
      Q::store(py + (long long)j * C, h, in && on0, in && on1);
      if ((m.end >> j & 1u) && fin != nullptr)
        store_state(fin, seq_index(p.q, b, t0 + j), C, c, c1, on0, on1, h);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(REC_THREADS)
recurrence_backward_kernel(SeqIn<T> x, SeqIn<T> u, SeqIn<T> v, const float *__restrict__ decay,
                           const float *__restrict__ initial, const float *__restrict__ ckpt, SeqIn<T> dy,
                           const float *__restrict__ dfin, T *__restrict__ dx, T *__restrict__ du, T *__restrict__ dv,
                           float *__restrict__ dinit, float *__restrict__ part, RecParams p) {
  using Q = Pair<T, VEC>;
  constexpr int L = REC_L, W = REC_W;
  __shared__ float4 agg[2][W][32];   // P, H of each warp's rows
  __shared__ float2 aggq[2][W][32];  // what leaves them towards earlier rows
  __shared__ float4 far[2][REC_MAX_CLUSTER][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = (int)(blockIdx.x % p.cs);
  const long long pair = blockIdx.x / p.cs;
  const int grp = (int)(pair % p.groups), b = (int)(pair / p.groups);
  const int C = p.q.C, c = Q::channel(grp, lane), c1 = VEC ? c + 1 : c + 32;
  const bool on0 = c < C, on1 = c1 < C;
  if (p.cs > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if (dinit != nullptr && rank == 0) empty_states(p, b, warp, dfin, dinit, c, c1, on0, on1);
  const float2 kz = make_float2(on0 ? p.scale * softplus(decay[c]) : 0.f,
                                on1 ? p.scale * softplus(decay[c1]) : 0.f);
  const bool series = __all_sync(0xffffffffu, kz.x <= REC_SERIES && kz.y <= REC_SERIES);
  const int tiles = ceil_div(p.q.T, REC_TILE), steps = ceil_div(tiles, p.cs);
  RowWalk walk;
  walk.init(p.q, b);
  float2 carry = f2(0.f), ddecay = f2(0.f);
  for (int it = steps - 1; it >= 0; --it) {
    const int tile = it * p.cs + rank, t0 = tile * REC_TILE + warp * L, half = it & 1;
    const RowMasks m = walk.masks<L>(p.q, t0);
    typename Q::Raw rx[L];
    float2 r[L], i[L], d[L], g[L];
    {
      typename Q::Raw ru[L], rv[L], rg[L];
      const T *px = x.row(b, t0) + c, *pu = u.row(b, t0) + c, *pv = v.row(b, t0) + c, *pg = dy.row(b, t0) + c;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const bool in = !(m.none >> j & 1u);
        rx[j] = Q::load(px + j * x.rs, in && on0, in && on1);
        ru[j] = Q::load(pu + j * u.rs, in && on0, in && on1);
        rv[j] = Q::load(pv + j * v.rs, in && on0, in && on1);
        rg[j] = Q::load(pg + j * dy.rs, in && on0, in && on1);
      }
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const Gates gt = gates(Q::get(ru[j]), Q::get(rv[j]), kz, series);
        r[j] = gt.r;
        i[j] = gt.i;
        d[j] = gt.d;
        g[j] = Q::get(rg[j]);
      }
    }
    float2 h = f2(0.f);
    if (tile < tiles) h = load_state(ckpt, (long long)b * tiles + tile, C, c, c1, on0, on1);
    const unsigned special = m.start | m.none;
    if (m.end != 0u && dfin != nullptr) {
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (m.end >> j & 1u)
          g[j] = add2(g[j], load_state(dfin, seq_index(p.q, b, t0 + j), C, c, c1, on0, on1));
    }
    // what the rows do to a state going down, and to a gradient going up
    auto input = [&](int j, float2 &q, float2 &rs) {
      q = beta_square2(d[j]);
      rs = make_float2(rsqf(q.x), rsqf(q.y));
      return mul2(i[j], Q::get(rx[j]));
    };
    float2 P = f2(1.f), H = f2(0.f), G = f2(0.f);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float2 q, rs;
      const float2 ix = input(j, q, rs);
      const float2 a = keep2(mul2(kz, r[j]), d[j], series);
      float2 bb = mul2(mul2(q, rs), ix);
      if (special >> j & 1u) {
        if (m.none >> j & 1u) bb = f2(0.f);
        else if (initial != nullptr)
          bb = fma2(a, load_state(initial, seq_index(p.q, b, t0 + j), C, c, c1, on0, on1), bb);
        P = f2(-1.f);
        H = bb;
      } else {
        P = special ? join(P, a) : mul2(P, a);
        H = fma2(a, H, bb);
      }
    }
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
      const float2 a = keep2(mul2(kz, r[j]), d[j], series);
      G = (special >> j & 1u) ? f2(0.f) : mul2(a, add2(g[j], G));
    }
    agg[half][warp][lane] = make_float4(P.x, P.y, H.x, H.y);
    aggq[half][warp][lane] = G;
    __syncthreads();
    float2 q = carry;
    if (p.cs > 1) {
      if (warp < p.cs) {
        float2 TP = f2(1.f), TG = f2(0.f);
#pragma unroll
        for (int k = W - 1; k >= 0; --k) {
          const float4 e = agg[half][k][lane];
          const float2 P2 = make_float2(e.x, e.y), G2 = aggq[half][k][lane];
          TG = apply(P2, G2, TG);
          TP = join(TP, P2);
        }
        store_peer(&far[half][rank][lane], warp, make_float4(TP.x, TP.y, TG.x, TG.y));
      }
      cluster_arrive();
      cluster_wait();
      for (int k = p.cs - 1; k >= 0; --k) {
        if (k == rank) q = carry;
        const float4 e = far[half][k][lane];
        carry = apply(make_float2(e.x, e.y), make_float2(e.z, e.w), carry);
      }
    }
#pragma unroll
    for (int k = W - 1; k >= 0; --k) {
      if (p.cs > 1 && k == warp) break;
      if (k == warp) carry = q;
      const float4 e = agg[half][k][lane];
      q = apply(make_float2(e.x, e.y), aggq[half][k][lane], q);
    }
    if (p.cs == 1) {
      const float2 next = q;
      q = carry;
      carry = next;
    }
    for (int k = 0; k < warp; ++k) {
      const float4 e = agg[half][k][lane];
      h = apply(make_float2(e.x, e.y), make_float2(e.z, e.w), h);
    }
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
      const float2 a = keep2(mul2(kz, r[j]), d[j], series);
      g[j] = add2(g[j], q);
      q = mul2(a, g[j]);
      if (special >> j & 1u) {
        if ((m.start >> j & 1u) && dinit != nullptr)
          store_state(dinit, seq_index(p.q, b, t0 + j), C, c, c1, on0, on1, q);
        q = f2(0.f);
      }
    }
    const long long at = ((long long)b * p.q.T + t0) * C + c;
    float2 sum = f2(0.f);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float2 bq, rs;
      const float2 ix = input(j, bq, rs);
      const float2 a = keep2(mul2(kz, r[j]), d[j], series), beta = mul2(bq, rs);
      if (special >> j & 1u) {
        h = f2(0.f);
        if ((m.start >> j & 1u) && initial != nullptr)
          h = load_state(initial, seq_index(p.q, b, t0 + j), C, c, c1, on0, on1);
        if (m.none >> j & 1u) g[j] = f2(0.f);
      }
      const float2 ddx = mul2(g[j], mul2(beta, i[j]));
      const float2 ddv = mul2(mul2(ddx, Q::get(rx[j])), add2(f2(1.f), neg2(i[j])));
      // dz / g = a (a / beta i x - h[t-1])
      const float2 dz = mul2(mul2(g[j], a), fma2(mul2(a, rs), ix, neg2(h)));
      const float2 z = mul2(kz, r[j]);
      const float2 ddu = mul2(mul2(dz, z), add2(f2(1.f), neg2(r[j])));
      sum = fma2(dz, r[j], sum);
      h = fma2(a, h, mul2(beta, ix));
      const bool in = t0 + j < p.q.T;
      Q::store(dx + at + (long long)j * C, ddx, in && on0, in && on1);
      Q::store(du + at + (long long)j * C, ddu, in && on0, in && on1);
      Q::store(dv + at + (long long)j * C, ddv, in && on0, in && on1);
    }
    ddecay = add2(ddecay, sum);
  }
  // this CTA's part of ddecay: the warps' sums in order
  __syncthreads();
  aggq[0][warp][lane] = ddecay;
  __syncthreads();
  if (warp == 0) {
    float2 s = aggq[0][0][lane];
#pragma unroll
    for (int k = 1; k < W; ++k) s = add2(s, aggq[0][k][lane]);
    store_state(part, (long long)b * p.cs + rank, C, c, c1, on0, on1, s);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(128)
recurrence_step_kernel(const T *__restrict__ x, long long xs, const T *__restrict__ u, long long us,
                       const T *__restrict__ v, long long vs, const float *__restrict__ decay,
                       float *__restrict__ state, T *__restrict__ y, RecParams p) {
  using Q = Pair<T, VEC>;
  const int lane = threadIdx.x & 31;
  const long long pair = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (pair >= (long long)p.groups * p.B) return;
  const int grp = (int)(pair % p.groups);
  const long long b = pair / p.groups;
  const int C = p.q.C, c = Q::channel(grp, lane), c1 = VEC ? c + 1 : c + 32;
  const bool on0 = c < C, on1 = c1 < C;
  const typename Q::Raw rx = Q::load(x + b * xs + c, on0, on1), ru = Q::load(u + b * us + c, on0, on1),
                        rv = Q::load(v + b * vs + c, on0, on1);
  const float2 h0 = load_state(state, b, C, c, c1, on0, on1);
  const float2 kz = make_float2(on0 ? p.scale * softplus(decay[c]) : 0.f,
                                on1 ? p.scale * softplus(decay[c1]) : 0.f);
  const Gates g = gates(Q::get(ru), Q::get(rv), kz, false);
  const float2 q = beta_square2(g.d);
  const float2 bb = mul2(mul2(q, make_float2(rsqf(q.x), rsqf(q.y))), mul2(g.i, Q::get(rx)));
  const float2 h = fma2(keep2(mul2(kz, g.r), g.d, false), h0, bb);
  store_state(state, b, C, c, c1, on0, on1, h);
  Q::store(y + b * C + c, h, on0, on1);
}

// ---- host --------------------------------------------------------------------------------------

// CTAs of a cluster along T: as many (a power of two, never more than there are tiles) as give every SM
// two CTAs.
inline int rec_cluster(const dwconv_b200_sequence &s) {
  const long long ctas = (long long)ceil_div(s.C, REC_GROUP) * s.B;
  const int tiles = ceil_div(s.T, REC_TILE);
  int cs = 1;
  while (cs < REC_MAX_CLUSTER && cs * 2 <= tiles && ctas * cs < 2 * 148) cs <<= 1;
  return cs;
}

inline RecParams rec_params(const dwconv_b200_sequence &s, float scale) {
  RecParams p;
  p.q = seq_list(s);
  p.B = s.B;
  p.groups = ceil_div(s.C, REC_GROUP);
  p.cs = rec_cluster(s);
  p.scale = scale;
  return p;
}

inline cudaLaunchConfig_t rec_config(const RecParams &p, cudaLaunchAttribute *attr, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)p.groups * p.B * p.cs));
  cfg.blockDim = dim3(REC_THREADS);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cs > 1 ? 1 : 0;
  return cfg;
}

struct RecArgs {
  const dwconv_b200_rows *x, *u, *v, *dy;
  const float *decay, *initial, *dfin;
  const float *ckpt_in;
  void *y, *dx, *du, *dv;
  float *fin, *ckpt, *dinit, *part;
  const dwconv_b200_sequence *s;
  float scale;
};

inline bool rec_vector(const RecArgs &a, size_t es) {
  const void *ptrs[] = {a.y, a.dx, a.du, a.dv};
  for (const void *q : ptrs)
    if (q != nullptr && !aligned_to(q, 2 * es)) return false;
  return a.s->C % 2 == 0 && rows_vector(*a.x, 2, es) && rows_vector(*a.u, 2, es) && rows_vector(*a.v, 2, es) &&
         (a.dy == nullptr || rows_vector(*a.dy, 2, es));
}

template <typename T, bool VEC> cudaError_t launch_forward(const RecArgs &a, cudaStream_t st) {
  const RecParams p = rec_params(*a.s, a.scale);
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = rec_config(p, attr, st);
  return cudaLaunchKernelEx(&cfg, recurrence_forward_kernel<T, VEC>, seq_in<T>(*a.x), seq_in<T>(*a.u),
                            seq_in<T>(*a.v), a.decay, a.initial, static_cast<T *>(a.y), a.fin, a.ckpt, p);
}
template <typename T, bool VEC> cudaError_t launch_backward(const RecArgs &a, cudaStream_t st) {
  const RecParams p = rec_params(*a.s, a.scale);
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = rec_config(p, attr, st);
  return cudaLaunchKernelEx(&cfg, recurrence_backward_kernel<T, VEC>, seq_in<T>(*a.x), seq_in<T>(*a.u),
                            seq_in<T>(*a.v), a.decay, a.initial, a.ckpt_in, seq_in<T>(*a.dy), a.dfin,
                            static_cast<T *>(a.dx), static_cast<T *>(a.du), static_cast<T *>(a.dv), a.dinit, a.part, p);
}

template <typename T> void forward_t(const RecArgs &a, cudaStream_t st) {
  if (rec_vector(a, sizeof(T))) launch_forward<T, true>(a, st);
  else launch_forward<T, false>(a, st);
}
template <typename T> void backward_t(const RecArgs &a, cudaStream_t st) {
  if (rec_vector(a, sizeof(T))) launch_backward<T, true>(a, st);
  else launch_backward<T, false>(a, st);
}

template <typename T>
void step_t(const void *x, long long xs, const void *u, long long us, const void *v, long long vs, const float *decay,
            float *state, void *y, const RecParams &p, cudaStream_t st) {
  const unsigned grid = (unsigned)ceil_div_ll((long long)p.groups * p.B, 4);
  const bool vec = p.q.C % 2 == 0 && xs % 2 == 0 && us % 2 == 0 && vs % 2 == 0 && aligned_to(x, 2 * sizeof(T)) &&
                   aligned_to(u, 2 * sizeof(T)) && aligned_to(v, 2 * sizeof(T)) && aligned_to(y, 2 * sizeof(T));
  if (vec)
    recurrence_step_kernel<T, true><<<grid, 128, 0, st>>>((const T *)x, xs, (const T *)u, us, (const T *)v, vs, decay,
                                                          state, (T *)y, p);
  else
    recurrence_step_kernel<T, false><<<grid, 128, 0, st>>>((const T *)x, xs, (const T *)u, us, (const T *)v, vs,
                                                           decay, state, (T *)y, p);
}

int check_recurrence(int dtype, const dwconv_b200_sequence *s) {
  if (!seq_dtype_ok(dtype)) return DWCONV_B200_UNSUPPORTED_DTYPE;
  const int e = check_sequence(s);
  if (e) return e;
  if ((long long)ceil_div(s->C, REC_GROUP) * s->B > ((1ll << 31) - 1) / REC_MAX_CLUSTER) return DWCONV_B200_TOO_LARGE;
  return DWCONV_B200_OK;
}

}  // namespace
}  // namespace dwb

using namespace dwb;

extern "C" {

size_t dwconv_b200_recurrence_checkpoint_bytes(const dwconv_b200_sequence *seq) {
  if (check_recurrence(DWCONV_B200_F32, seq) != DWCONV_B200_OK) return 0;
  const size_t n = (size_t)seq->B * ceil_div(seq->T, REC_TILE) * seq->C * sizeof(float);
  return (n + 15) / 16 * 16 + 16;
}

size_t dwconv_b200_recurrence_workspace_bytes(const dwconv_b200_sequence *seq) {
  if (check_recurrence(DWCONV_B200_F32, seq) != DWCONV_B200_OK) return 0;
  const size_t n = (size_t)seq->B * rec_cluster(*seq) * seq->C * sizeof(float);
  return (n + 15) / 16 * 16 + 16;
}

int dwconv_b200_recurrence(const dwconv_b200_rows *x, const dwconv_b200_rows *u, const dwconv_b200_rows *v,
                           const float *decay, const float *initial, void *y, float *final_state, float *checkpoints,
                           int dtype, const dwconv_b200_sequence *seq, float scale, void *stream) {
  int e = check_recurrence(dtype, seq);
  if (e) return e;
  const size_t es = elem_size(dtype);
  if ((e = check_rows(x, es)) != 0 || (e = check_rows(u, es)) != 0 || (e = check_rows(v, es)) != 0) return e;
  if (decay == nullptr || y == nullptr || !(scale > 0.f)) return DWCONV_B200_BAD_ARGUMENT;
  if (!aligned_to(decay, 4) || !aligned_to(y, es) || (initial && !aligned_to(initial, 4)) ||
      (final_state && !aligned_to(final_state, 4)) || (checkpoints && !aligned_to(checkpoints, 16)))
    return DWCONV_B200_MISALIGNED;
  RecArgs a{};
  a.x = x; a.u = u; a.v = v; a.decay = decay; a.initial = initial; a.y = y; a.fin = final_state;
  a.ckpt = checkpoints; a.s = seq; a.scale = scale;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: forward_t<float>(a, st); break;
    case DWCONV_B200_F16: forward_t<__half>(a, st); break;
    default: forward_t<__nv_bfloat16>(a, st); break;
  }
  return api_launch_status();
}

int dwconv_b200_recurrence_backward(const dwconv_b200_rows *x, const dwconv_b200_rows *u, const dwconv_b200_rows *v,
                                    const float *decay, const float *initial, const float *checkpoints,
                                    const dwconv_b200_rows *dy, const float *dfinal, void *dx, void *du, void *dv,
                                    float *ddecay, float *dinitial, void *workspace, size_t workspace_bytes, int dtype,
                                    const dwconv_b200_sequence *seq, float scale, void *stream) {
  int e = check_recurrence(dtype, seq);
  if (e) return e;
  const size_t es = elem_size(dtype);
  if ((e = check_rows(x, es)) != 0 || (e = check_rows(u, es)) != 0 || (e = check_rows(v, es)) != 0 ||
      (e = check_rows(dy, es)) != 0)
    return e;
  if (decay == nullptr || checkpoints == nullptr || dx == nullptr || du == nullptr || dv == nullptr ||
      ddecay == nullptr || workspace == nullptr || !(scale > 0.f))
    return DWCONV_B200_BAD_ARGUMENT;
  if (!aligned_to(decay, 4) || !aligned_to(checkpoints, 16) || !aligned_to(dx, es) || !aligned_to(du, es) ||
      !aligned_to(dv, es) || !aligned_to(ddecay, 4) || (initial && !aligned_to(initial, 4)) ||
      (dfinal && !aligned_to(dfinal, 4)) || (dinitial && !aligned_to(dinitial, 4)) || !aligned_to(workspace, 16))
    return DWCONV_B200_MISALIGNED;
  if (workspace_bytes < dwconv_b200_recurrence_workspace_bytes(seq)) return DWCONV_B200_WORKSPACE_TOO_SMALL;
  RecArgs a{};
  a.x = x; a.u = u; a.v = v; a.dy = dy; a.decay = decay; a.initial = initial; a.dfin = dfinal;
  a.ckpt_in = checkpoints; a.dx = dx; a.du = du; a.dv = dv; a.dinit = dinitial;
  a.part = static_cast<float *>(workspace); a.s = seq; a.scale = scale;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: backward_t<float>(a, st); break;
    case DWCONV_B200_F16: backward_t<__half>(a, st); break;
    default: backward_t<__nv_bfloat16>(a, st); break;
  }
  e = api_launch_status();
  if (e) return e;
  launch_column_sum(a.part, (long long)seq->B * rec_cluster(*seq), seq->C,
                    ColumnSumOut{ddecay, nullptr, DWCONV_B200_F32, seq->C, 1, decay, scale}, st);
  return api_launch_status();
}

int dwconv_b200_recurrence_step(const void *x, long long x_stride, const void *u, long long u_stride, const void *v,
                                long long v_stride, const float *decay, float *state, void *y, int dtype, int B, int C,
                                float scale, void *stream) {
  const dwconv_b200_sequence s{B, 1, C, nullptr, 0};
  const int e = check_recurrence(dtype, &s);
  if (e) return e;
  if (x == nullptr || u == nullptr || v == nullptr || decay == nullptr || state == nullptr || y == nullptr ||
      !(scale > 0.f))
    return DWCONV_B200_BAD_ARGUMENT;
  const size_t es = elem_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(u, es) || !aligned_to(v, es) || !aligned_to(decay, 4) ||
      !aligned_to(state, 4) || !aligned_to(y, es))
    return DWCONV_B200_MISALIGNED;
  const RecParams p = rec_params(s, scale);
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: step_t<float>(x, x_stride, u, u_stride, v, v_stride, decay, state, y, p, st); break;
    case DWCONV_B200_F16: step_t<__half>(x, x_stride, u, u_stride, v, v_stride, decay, state, y, p, st); break;
    default: step_t<__nv_bfloat16>(x, x_stride, u, u_stride, v, v_stride, decay, state, y, p, st); break;
  }
  return api_launch_status();
}

}  // extern "C"
