// Gated linear recurrence over [B, T, C] sequences: a scan along T with its gates computed on the
// way, the backward pass, and the one-row step (declarations: include/dwconv_b200.h).
//
//   r = sigmoid(u), i = sigmoid(v), z = k r with k = scale softplus(decay)
//   a = exp(-z),  beta = sqrt(1 - a^2),  h[t] = a h[t-1] + beta i x,  y = h
// and with g[t] = dy[t] + a[t+1] g[t+1], rho = z / beta:
//   dx = g beta i,  dv = dx x (1 - i),  dz z = g a (a i x rho - z h[t-1]),  du = dz z (1 - r),
//   ddecay = sigmoid(decay) / softplus(decay) sum_t dz z,  dinitial = a[0] g[0].
// For the long memories such models use z is small.  There a = 1 + (exp(-z) - 1) comes from the power
// series of the bracket, and with t = sqrt(r) = rsqrt(1 + exp(-u))
//   beta = sqrt(2 k) t p(z),  rho = sqrt(k / 2) t / p(z),  p(z) = sqrt((1 - exp(-2 z)) / (2 z)),
// p and 1 / p by their power series: no difference of nearly equal numbers, and two special-function
// calls per gate (the special-function unit is one of the three things that bound these kernels, beside
// memory and the issue of instructions).
//
// Bound by memory: forward x, u, v in and y out; backward x, u, v, dy in and dx, du, dv out.
//
// Layout.  A lane owns two channels, a warp 64 channels of L consecutive rows, a CTA of W warps a tile
// of W * L rows.  A warp reduces its rows to one pair (P, H): the state that leaves them is
// P h + H.  Pairs meet in shared memory, every warp folds those in front of it onto the state that
// enters the tile, and walks its rows once more from registers.  Tiles follow one another along T.
// Where there are too few (channel block, batch) pairs to fill the device evenly, a cluster of CTAs takes
// neighbouring tiles together and passes its tiles' pairs on by asynchronous stores to distributed
// shared memory, which signal the receiving CTA's barrier themselves (a cluster-wide barrier with its
// memory fence cost a fifth of the time): no second pass over the data, and the same order of operations
// on every run.
//
// A warp has the rows of its next tile copied to shared memory by tensor copies (TMA, one box of L rows
// by 64 channels per tensor; what lies outside the tensor arrives as zeros) as soon as those of the
// current one are in registers, so that the barriers, folds and stores run under them.  Tensors that the
// copy engine cannot address (rows off 16-byte boundaries) are read two elements per lane instead, without
// copies ahead.
//
// The forward pass keeps the fp32 state that enters every 32nd row; the backward pass starts from it, so it
// reads y nowhere and its h[t-1] have not been rounded to the data's type.
//
// Measured (bf16, 8 x 8192 rows of 4096 channels): forward 432 us, 5.0 TB/s; backward 893 us, 4.2 TB/s.  Neither
// memory (76 % and 64 % of a copy's rate) nor the issue of instructions (58 % and 57 % of the slots, with 74 and 146
// per warp and row) is full: what is left is the latency of a tile's steps, one after another, which 23 and 14
// active warps per SM do not cover.  Where some channel of a CTA decays faster (scale softplus(decay) above REC_SERIES) the
// exponential takes the series' place: 559 and 1049 us with decays from 0.3 to 0.999; 4 x 2048 rows of 2048: 43 and
// 84 us, then 53 and 96.  Rows that the copy engine cannot address (2047 channels): 74 and 160.
#include <atomic>
#include <cmath>

#include "rows_engine.cuh"
#include "seq_common.cuh"
#include "tensor_map.cuh"

namespace dwb {
namespace {

__device__ int g_seq_error_flag;  // raised by a wait that ran out

constexpr int REC_L = 8;       // rows of a warp
constexpr int REC_GROUP = 64;  // channels of a warp
constexpr int REC_CKPT = 32;   // rows between the states that are kept for the backward pass
constexpr int REC_MAX_CLUSTER = 16;  // more than 8 needs the non-portable attribute
// Largest z for which the power series are used: what they omit is 5e-8 of exp(-z) - 1 and 2e-9 of p there.
constexpr float REC_SERIES = 0.125f;

// ---- arithmetic on channel pairs ---------------------------------------------------------------

// The same value, of which the compiler does not know that: what is computed from it again is not kept in
// a register meanwhile.
__device__ __forceinline__ void forget(float2 &v) { asm volatile("" : "+f"(v.x), "+f"(v.y)); }

__device__ __forceinline__ float2 root_sigmoid2(float2 v) {
  const float2 s = one_plus_exp2(v);
  return make_float2(rsqf(s.x), rsqf(s.y));
}

__device__ __forceinline__ float2 horner2(float2 p, float2 s, float c) { return fma2(p, s, f2(c)); }
// exp(s) - 1, p(-s) and 1 / p(-s) for -REC_SERIES <= s <= 0, from the Taylor expansions of
// exp(s), exp(s / 2) sqrt(sinh(s) / s) and its reciprocal about 0.
__device__ __forceinline__ float2 expm1_series2(float2 s) {
  float2 p = horner2(f2(1.f / 120.f), s, 1.f / 24.f);
  p = horner2(p, s, 1.f / 6.f);
  p = horner2(p, s, 0.5f);
  return mul2(s, horner2(p, s, 1.f));
}
__device__ __forceinline__ float2 p_series2(float2 s) {
  float2 p = horner2(f2(3.f / 1280.f), s, 79.f / 5760.f);
  p = horner2(p, s, 1.f / 16.f);
  p = horner2(p, s, 5.f / 24.f);
  p = horner2(p, s, 0.5f);
  return horner2(p, s, 1.f);
}
__device__ __forceinline__ float2 inverse_p_series2(float2 s) {
  float2 p = horner2(f2(-19.f / 11520.f), s, -1.f / 640.f);
  p = horner2(p, s, 1.f / 48.f);
  p = horner2(p, s, 1.f / 24.f);
  p = horner2(p, s, -0.5f);
  return horner2(p, s, 1.f);
}

// What a lane keeps of its channels: -k and sqrt(2 k).
struct Rate {
  float2 ks, root;
};

// 1 - a^2 for any s, kept off zero so that its reciprocal root stays finite (z = 0: closed gate).
__device__ __forceinline__ float2 beta_square2(float2 s) {
  float2 m = expm1_series2(s);
  const float2 e = mul2(s, f2(LOG2E));
  if (!(s.x >= -REC_SERIES)) m.x = ex2f(e.x) - 1.f;
  if (!(s.y >= -REC_SERIES)) m.y = ex2f(e.y) - 1.f;
  const float2 t = fma2(m, m, add2(m, m));
  float2 r;  // a NaN stays one
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r.x) : "f"(-t.x), "f"(1e-37f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r.y) : "f"(-t.y), "f"(1e-37f));
  return r;
}
__device__ __forceinline__ float2 rsq2(float2 q) { return make_float2(rsqf(q.x), rsqf(q.y)); }

// a = exp(s).  By the series good to a unit or two in its own last place; below -REC_SERIES, which SERIES rules out
// for this CTA's channels, s log2(e) is rounded before the exponential, whose relative error grows by 6e-8 per
// unit of |s| (absolutely it stays below 3e-8).
template <bool SERIES> __device__ __forceinline__ float2 keep2(float2 s) {
  float2 a = add2(expm1_series2(s), f2(1.f));
  if constexpr (!SERIES) {
    const float2 e = mul2(s, f2(LOG2E));
    if (!(s.x >= -REC_SERIES)) a.x = ex2f(e.x);
    if (!(s.y >= -REC_SERIES)) a.y = ex2f(e.y);
  }
  return a;
}
template <bool SERIES> __device__ __forceinline__ float2 beta2(float2 t, float2 s, const Rate &k) {
  if constexpr (SERIES) return mul2(mul2(t, k.root), p_series2(s));
  const float2 q = beta_square2(s);
  return mul2(q, rsq2(q));
}
template <bool SERIES> __device__ __forceinline__ float2 rho2(float2 t, float2 s, const Rate &k) {
  if constexpr (SERIES) return mul2(mul2(t, mul2(k.root, f2(0.5f))), inverse_p_series2(s));
  const float2 r = mul2(s, rsq2(beta_square2(s)));
  return make_float2(-r.x, -r.y);
}

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v : log1pf(expf(v)); }

// ---- channel pairs of a lane -------------------------------------------------------------------

// VEC: channels c, c + 1, one load.  Otherwise (odd C, odd strides) channels c0 and c1 = c0 + 32, one each.
// Lanes beyond the last channel work on the last one too, and store the same values to the same places:
// no access needs a test.
struct Chan {
  int c0, c1;
};
template <typename T, bool VEC> struct Pair;
template <typename T> struct Pair<T, true> {
  using P = Pack<T, 2>;
  using Raw = typename P::Raw;
  static __device__ __forceinline__ Chan channels(int g, int lane, int C) {
    const int c = min(g * REC_GROUP + 2 * lane, C - 2);
    return Chan{c, c + 1};
  }
  static __device__ __forceinline__ Raw zero() { return P::zero(); }
  static __device__ __forceinline__ Raw closed() {
    const float f[2] = {-__int_as_float(0x7f800000), -__int_as_float(0x7f800000)};
    return P::pack(f);
  }
  static __device__ __forceinline__ Raw load(const T *row, const Chan &c) { return P::load(row + c.c0); }
  static __device__ __forceinline__ float2 get(const Raw &r) {
    float f[2];
    P::unpack(r, f);
    return make_float2(f[0], f[1]);
  }
  static __device__ __forceinline__ void store(T *row, const Chan &c, float2 v) {
    const float f[2] = {v.x, v.y};
    P::store(row + c.c0, P::pack(f));
  }
};
template <typename T> struct Pair<T, false> {
  struct Raw { T a, b; };
  static __device__ __forceinline__ Chan channels(int g, int lane, int C) {
    return Chan{min(g * REC_GROUP + lane, C - 1), min(g * REC_GROUP + lane + 32, C - 1)};
  }
  static __device__ __forceinline__ Raw zero() { return Raw{Elem<T>::from_acc(0.f), Elem<T>::from_acc(0.f)}; }
  static __device__ __forceinline__ Raw closed() {
    const T inf = Elem<T>::from_acc(-__int_as_float(0x7f800000));
    return Raw{inf, inf};
  }
  static __device__ __forceinline__ Raw load(const T *row, const Chan &c) { return Raw{row[c.c0], row[c.c1]}; }
  static __device__ __forceinline__ float2 get(const Raw &r) {
    return make_float2(Elem<T>::to_acc(r.a), Elem<T>::to_acc(r.b));
  }
  static __device__ __forceinline__ void store(T *row, const Chan &c, float2 v) {
    row[c.c0] = Elem<T>::from_acc(v.x);
    row[c.c1] = Elem<T>::from_acc(v.y);
  }
};

// ---- copies ahead ------------------------------------------------------------------------------

struct RecMaps {
  CUtensorMap m[4];  // x, u, v (, dy) as (channel, row, batch)
};
__device__ __forceinline__ void rows_load(void *to, const CUtensorMap *map, int c, int t, int b, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(to)),
      "l"(map), "r"(c), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}
// What became of a CTA's waits (beside the barriers, in shared memory).
struct RecWaits {
  int give_up;    // from this iteration on the CTA has no part in the cluster's exchange
  int stuck[8];   // by warp: 0, or 1 + the parity of the copies that it waited for in vain
  int sent[16];   // by rank, at the end: the iterations whose pairs that CTA has sent
};
__device__ __forceinline__ int look_at(const int &word) { return *(const volatile int *)&word; }
__device__ __forceinline__ bool mbar_test_wait(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded waits.  One that runs out raises the flag that dwconv_b200_device_status reports; the kernel goes on to its
// end, but a barrier whose phase is not complete is not armed again: a warp copies no more rows ahead, or the CTA has
// no more part in its cluster's exchange (nor waits for it again).  (The waits acquire at CTA scope: what they wait
// for lies in this CTA's shared memory, counted by the barrier as it arrives.  At cluster scope every poll would throw
// the L1 cache away as well.)  Lanes poll for themselves: any that fails says so, in front of the warp's or the CTA's
// next barrier.
__device__ __forceinline__ bool wait_polls(uint64_t *bar, uint32_t parity, unsigned polls) {
  for (unsigned i = 0; i < polls; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ void wait_copies(uint64_t *bar, uint32_t parity, unsigned polls, int &stuck) {
  if (mbar_test_wait(bar, parity) || look_at(stuck) != 0 || wait_polls(bar, parity, polls)) return;
  atomicExch(&g_seq_error_flag, 8);
  stuck = 1 + (int)parity;
}
__device__ __forceinline__ void wait_peers(uint64_t *bar, int iteration, unsigned polls, int &give_up) {
  if (wait_polls(bar, iteration >> 1 & 1, polls)) return;
  atomicExch(&g_seq_error_flag, 8);
  atomicMin(&give_up, iteration + 1);
}

// Rows at T and behind: a gate of -infinity is closed, the state passes through it.  Every lane
// writes what it reads itself (the same as others that share its channels).
template <typename T> __device__ __forceinline__ void close_rows(T *gate, int rows, int col) {
#pragma unroll
  for (int j = 0; j < REC_L; ++j)
    if (j >= rows) Pack<T, 2>::store(gate + j * REC_GROUP + col, Pair<T, true>::closed());
}

// ---- rows of a warp ----------------------------------------------------------------------------

// Which of a warp's L rows begin a sequence, end one, or belong to none (bit j: row t0 + j).
// start_seq, end_seq: the sequence of the last row of each kind.
struct RowMasks {
  unsigned start, end, none;
  int start_seq, end_seq;
};

// For packed sequences: spans one after the other, starting from the one that the warp's last tile ended in.
struct RowWalk {
  SeqSpan sp{-1, 0, 0};
  template <int L> __device__ __forceinline__ RowMasks masks(const SeqList &q, int t0) {
    RowMasks m{0u, 0u, 0u, -1, -1};
    int t = t0;
    const int end = min(t0 + L, q.T);
    while (t < end) {
      if (!(t >= sp.begin && t < sp.next)) sp = seq_locate(q, t);
      const int to = min(sp.next, end);
      if (sp.seq < 0) {
        m.none |= (1u << (to - t0)) - (1u << (t - t0));
      } else {
        if (t == sp.begin) {
          m.start |= 1u << (t - t0);
          m.start_seq = sp.seq;
        }
        if (to == sp.next) {
          m.end |= 1u << (to - 1 - t0);
          m.end_seq = sp.seq;
        }
      }
      t = to;
    }
    t = max(t, t0);
    if (t < t0 + L) m.none |= (1u << L) - (1u << (t - t0));  // at T and behind
    return m;
  }
};

// The sequence of row t0 + j, one of those in `mask`, of which `last` is the sequence of the last one.
__device__ __forceinline__ int seq_of(const SeqList &q, int t0, int j, unsigned mask, int last) {
  return mask >> j == 1u ? last : seq_locate(q, t0 + j).seq;
}

__device__ __forceinline__ float2 load_state(const float *s, long long j, int C, const Chan &c) {
  return make_float2(s[j * C + c.c0], s[j * C + c.c1]);
}
__device__ __forceinline__ void store_state(float *s, long long j, int C, const Chan &c, float2 v) {
  s[j * C + c.c0] = v.x;
  s[j * C + c.c1] = v.y;
}

// Folding pairs.  PACKED: a pair whose rows begin a sequence takes nothing from in front of it, whatever
// stands there (an infinity times zero would not be zero): its P is -1, which no product of decays is, and
// stays -1 whatever it is multiplied by (a NaN would take the sign away).
__device__ __forceinline__ bool cut(float2 P) { return __float_as_int(P.x) < 0; }
template <bool PACKED> __device__ __forceinline__ float2 join(float2 P, float2 Q) {
  return PACKED && (cut(P) || cut(Q)) ? f2(-1.f) : mul2(P, Q);
}
template <bool PACKED> __device__ __forceinline__ float2 apply(float2 P, float2 H, float2 h) {
  return PACKED && cut(P) ? H : fma2(P, h, H);
}

// (P, H) of warps from .. to - 1 of a tile, onto what stands in (P, H).
template <bool PACKED, int W>
__device__ __forceinline__ void fold(const float4 (&agg)[W][32], int lane, int from, int to, float2 &P, float2 &H) {
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < from || w >= to) continue;
    const float4 e = agg[w][lane];
    const float2 P2 = make_float2(e.x, e.y), H2 = make_float2(e.z, e.w);
    H = apply<PACKED>(P2, H2, H);
    P = join<PACKED>(P, P2);
  }
}

// ---- thread-block clusters ---------------------------------------------------------------------

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 16 bytes to the same place of a peer's shared memory, counted by the same barrier of the peer.
__device__ __forceinline__ void store_peer(const void *mine, const uint64_t *bar, int rank, float4 v) {
  uint32_t a, m;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(a), "f"(v.x),
      "f"(v.y), "f"(v.z), "f"(v.w), "r"(m)
      : "memory");
}

// The bytes of which no store will tell this CTA's barrier.
__device__ __forceinline__ void complete_tx(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void store_peer_word(const int *mine, int rank, int v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

// The end of a cluster's walk, for every thread of it: no CTA leaves before its peers have sent it all they
// will, nor, where a wait ran out, before that has landed.
// A CTA sends the pairs of iteration n only where it has all pairs of n - 1.  One that gives up before iteration n has
// sent those of n - 1, for which its barrier still waits, and its peers may have sent theirs of n, for which it has
// not armed its barrier; nobody can have sent more.
__device__ __forceinline__ void leave_cluster(RecWaits *waits, uint64_t *met, int cs, int rank, int steps) {
  __syncthreads();
  const int n = waits->give_up;
  if (threadIdx.x < cs) store_peer_word(&waits->sent[rank], threadIdx.x, min(n, steps));
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (n > steps || threadIdx.x != 0) return;
  uint32_t missing = 0, ahead = 0;
  for (int r = 0; r < cs; ++r) {
    missing += waits->sent[r] < n ? 512 : 0;
    ahead += waits->sent[r] > n ? 512 : 0;
  }
  uint64_t *bar = met + ((n - 1) & 1), *next = met + (n & 1);
  if (missing > 0) complete_tx(bar, missing);
  (void)mbar_wait_bounded(bar, (n - 1) >> 1 & 1);
  if (ahead == 0) return;
  mbar_arrive_expect_tx(next, ahead);
  (void)mbar_wait_bounded(next, n >> 1 & 1);
}
// The end of a warp's walk: copies that it waited for in vain land before the CTA's shared memory is another's.
__device__ __forceinline__ void land_copies(uint64_t *bar, const int &stuck) {
  const int s = look_at(stuck);
  if (s != 0) (void)mbar_wait_bounded(bar, s - 1);
}

// The warp's number, known to the compiler to be the same in all its lanes.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0); }

struct RecParams {
  SeqList q;
  int B, groups, cs;  // cs: CTAs of a cluster
  float scale;
  unsigned polls;  // of a wait, before it has run out
  int leaver;      // -1, or the rank of a CTA that gives up before iteration 1 (dwconv_b200_debug_expire)
};

// Sequences without a row: what enters leaves.
template <int W>
__device__ __forceinline__ void empty_states(const RecParams &p, int warp, const float *from, float *to, const Chan &c) {
  for (int j = warp; j < p.q.S; j += W)
    if (seq_bound(p.q, j) >= seq_bound(p.q, j + 1))
      store_state(to, j, p.q.C, c, from ? load_state(from, j, p.q.C, c) : f2(0.f));
}

// Shared memory of a CTA of W warps: the rows of NT tensors (FAST), barriers, the pairs of the warps for two
// tiles, what enters the CTA's tile (two), backward the rows' decays, the pairs of the cluster for two tiles, PACKED the first offsets.
template <typename T> constexpr int rec_stage(int W, int NT) { return W * REC_L * REC_GROUP * NT * (int)sizeof(T); }
constexpr int REC_BARRIERS = 256;  // one per warp for its copies, two for the cluster's pairs; from 128 on RecWaits
constexpr int REC_OFFSETS = 1024;  // as many offsets of packed sequences are kept in shared memory
constexpr int rec_smem(int W, int stage, bool backward, bool packed, int cs) {
  return stage + (packed ? REC_OFFSETS * 4 : 0) + (backward ? 0 : 2 * 32 * 8) + REC_BARRIERS + 2 * W * 32 * (backward ? 24 : 16) + (backward ? W * REC_L * REC_GROUP * 4 : 0) +
         (cs > 1 ? 2 * cs * 32 * 16 : 0);
}

// The list's offsets in shared memory, where they fit.
__device__ __forceinline__ void keep_offsets(SeqList &q, int *kept) {
  if (q.S + 1 > REC_OFFSETS) return;
  for (int j = threadIdx.x; j <= q.S; j += blockDim.x) kept[j] = q.offsets[j];
  __syncthreads();
  q.offsets = kept;
}

// Barriers of a CTA; with clusters, a peer's shared memory may be written once the peer has passed here.
template <int W, bool FAST>
__device__ __forceinline__ void start_cta(uint64_t *bars, RecWaits *waits, const RecParams &p, int rank) {
  if (!FAST && p.cs == 1) return;
  if (threadIdx.x == 0) {
    waits->give_up = rank == p.leaver ? 1 : 0x7fffffff;
    for (int n = 0; n < W; ++n) waits->stuck[n] = 0;
    for (int n = 0; n < W + 2; ++n) mbar_init(bars + n, 1);
    fence_barrier_init();
  }
  __syncthreads();
  if (p.cs > 1) {
    cluster_arrive();
    cluster_wait();
  }
}

// FAST: rows copied ahead by tensor copies; otherwise read where they are used, channels c and c + 32 per lane.
//
// Pairs have two places each, for even and odd tiles: a warp writes those of tile n + 2 behind tile n + 1's
// barrier, which every warp reaches done with tile n; a peer sends those of tile n + 2 once it has this CTA's
// of tile n + 1, which this CTA sends behind the same barrier.
template <typename T, int W, bool FAST, bool PACKED, bool SERIES>
__device__ __forceinline__ void forward_body(const RecMaps &maps, SeqIn<T> x, SeqIn<T> u, SeqIn<T> v,
                                             const float *__restrict__ initial, T *__restrict__ y,
                                             float *__restrict__ fin, float *__restrict__ ckpt, const RecParams &p,
                                             const Rate &k) {
  using Q = Pair<T, FAST>;
  constexpr int L = REC_L, NT = 3, TILE = W * L;
  extern __shared__ __align__(128) unsigned char smem[];
  T *stage = reinterpret_cast<T *>(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (FAST ? rec_stage<T>(W, NT) : 0)), *met = bars + W;
  RecWaits *waits = reinterpret_cast<RecWaits *>(bars + 16);
  float4(*agg)[W][32] = reinterpret_cast<float4(*)[W][32]>(reinterpret_cast<unsigned char *>(bars) + REC_BARRIERS);
  float2(*entry)[32] = reinterpret_cast<float2(*)[32]>(agg + 2);  // [2]: the state that enters the CTA's tile
  float4 *far = reinterpret_cast<float4 *>(entry + 2);            // [2][cs][32]
  const int lane = threadIdx.x & 31, warp = uniform_warp();
  const int rank = (int)(blockIdx.x % p.cs);
  const long long pair = blockIdx.x / p.cs;
  const int grp = (int)(pair % p.groups), b = (int)(pair / p.groups);
  const int C = p.q.C;
  const Chan c = Q::channels(grp, lane, C);
  const int tiles = ceil_div(p.q.T, TILE), steps = ceil_div(tiles, p.cs);
  T *mine = stage + warp * (NT * L * REC_GROUP);
  const int col = c.c0 - grp * REC_GROUP;  // of this lane in the staged rows
  auto start_copies = [&](int tile) {
    if (lane == 0 && look_at(waits->stuck[warp]) == 0) {
      const int t = tile * TILE + warp * L;
      mbar_arrive_expect_tx(bars + warp, NT * L * REC_GROUP * (uint32_t)sizeof(T));
#pragma unroll
      for (int n = 0; n < NT; ++n) rows_load(mine + n * L * REC_GROUP, &maps.m[n], grp * REC_GROUP, t, b, bars + warp);
    }
  };
  SeqList q = p.q;
  if (PACKED) {
    int *kept = reinterpret_cast<int *>(far + (p.cs > 1 ? 2 * p.cs * 32 : 0));
    keep_offsets(q, kept);
  }
  start_cta<W, FAST>(bars, waits, p, rank);
  if (FAST && steps > 0) start_copies(rank);
  if (PACKED && fin != nullptr && rank == 0) empty_states<W>(p, warp, initial, fin, c);
  RowWalk walk;
  float2 carry = f2(0.f);
  if (!PACKED && initial != nullptr) carry = load_state(initial, b, C, c);

  RowMasks next_m{0u, 0u, 0u, -1, -1};
  float2 next_entry = f2(0.f);  // the state that the last sequence to begin in the warp's rows begins with
  auto look = [&](int t) {
    next_m = walk.masks<L>(q, t);
    if (next_m.start != 0u && initial != nullptr) next_entry = load_state(initial, next_m.start_seq, C, c);
  };
  if (PACKED && steps > 0) look(rank * TILE + warp * L);
  for (int it = 0; it < steps; ++it) {
    const int tile = it * p.cs + rank, t0 = tile * TILE + warp * L, rows = p.q.T - t0, half = it & 1;
    float2 a[L], bb[L];
    const RowMasks m = next_m;
    const float2 first = next_entry;
    {
      typename Q::Raw rx[L], ru[L], rv[L];
      if constexpr (FAST) {
        wait_copies(bars + warp, it & 1, p.polls, waits->stuck[warp]);
        if (!PACKED && rows < L) close_rows<T>(mine + L * REC_GROUP, rows, col);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          rx[j] = Q::P::load(mine + j * REC_GROUP + col);
          ru[j] = Q::P::load(mine + (L + j) * REC_GROUP + col);
          rv[j] = Q::P::load(mine + (2 * L + j) * REC_GROUP + col);
        }
      } else {
        const T *px = x.row(b, t0), *pu = u.row(b, t0), *pv = v.row(b, t0);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          rx[j] = j < rows ? Q::load(px + j * x.rs, c) : Q::zero();
          ru[j] = j < rows ? Q::load(pu + j * u.rs, c) : Q::zero();
          if (!PACKED && j >= rows) ru[j] = Q::closed();
          rv[j] = j < rows ? Q::load(pv + j * v.rs, c) : Q::zero();
        }
      }
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const float2 t = root_sigmoid2(Q::get(ru[j])), s = mul2(k.ks, mul2(t, t));
        a[j] = keep2<SERIES>(s);
        bb[j] = mul2(beta2<SERIES>(t, s, k), mul2(sigmoid2(Q::get(rv[j])), Q::get(rx[j])));
      }
    }
    if constexpr (FAST) {
      __syncwarp();
      if (it + 1 < steps) start_copies(tile + p.cs);
    }
    float2 P = f2(1.f), H = f2(0.f);
    if (!PACKED || (m.start | m.none) == 0u) {
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
            bb[j] = fma2(a[j], (m.start >> j == 1u ? first : load_state(initial, seq_locate(q, t0 + j).seq, C, c)), bb[j]);
          P = f2(-1.f);
          H = bb[j];
        } else {
          P = join<PACKED>(P, a[j]);
          H = fma2(a[j], H, bb[j]);
        }
      }
    }
    agg[half][warp][lane] = make_float4(P.x, P.y, H.x, H.y);
    bool cuts = false;  // whether a sequence begins in this CTA's tile
    if (PACKED) cuts = __syncthreads_or((int)(m.start | m.none));
    else __syncthreads();
    const bool part = p.cs > 1 && look_at(waits->give_up) > it;
    if (p.cs > 1 && warp < p.cs) {
      // the CTA's pair, folded by each of the warps that pass it on
      float2 TP = f2(1.f), TH = f2(0.f);
      if (cuts) fold<PACKED, W>(agg[half], lane, 0, W, TP, TH);
      else fold<false, W>(agg[half], lane, 0, W, TP, TH);
      float4 *there = far + (half * p.cs + rank) * 32 + lane;
      if (part) {
        for (int peer = warp; peer < p.cs; peer += W)
          store_peer(there, met + half, peer, make_float4(TP.x, TP.y, TH.x, TH.y));
        if (threadIdx.x == 0) mbar_arrive_expect_tx(met + half, p.cs * 512);
      }
    }
    float2 h = carry;
    if (p.cs > 1) {
      // this CTA's rows in front of the warp's, while the peers' pairs are on their way
      float2 FP = f2(1.f), FH = f2(0.f);
      if (cuts) fold<PACKED, W>(agg[half], lane, 0, warp, FP, FH);
      else fold<false, W>(agg[half], lane, 0, warp, FP, FH);
      if (PACKED && it + 1 < steps) look(t0 + p.cs * TILE);
      if (warp == 0) {  // one warp waits for the peers' pairs and folds them for all
        if (part) wait_peers(met + half, it, p.polls, waits->give_up);
        for (int w = 0; w < p.cs; ++w) {
          if (w == rank) entry[half][lane] = carry;
          const float4 e = far[(half * p.cs + w) * 32 + lane];
          carry = apply<PACKED>(make_float2(e.x, e.y), make_float2(e.z, e.w), carry);
        }
      }
      __syncthreads();
      h = apply<PACKED>(FP, FH, entry[half][lane]);
    } else {
      float2 in = h;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w == warp) in = h;
        const float4 e = agg[half][w][lane];
        h = apply<PACKED>(make_float2(e.x, e.y), make_float2(e.z, e.w), h);
      }
      carry = h;
      h = in;
      if (PACKED && it + 1 < steps) look(t0 + TILE);
    }
    if (ckpt != nullptr && warp * L % REC_CKPT == 0 && rows > 0)
      store_state(ckpt, (long long)b * ceil_div(p.q.T, REC_CKPT) + t0 / REC_CKPT, C, c, h);
    T *py = y + ((long long)b * p.q.T + t0) * C;
    if (rows >= L && (!PACKED || (m.start | m.none | m.end) == 0u)) {
#pragma unroll
      for (int j = 0; j < L; ++j) {
        h = fma2(a[j], h, bb[j]);
        Q::store(py + (long long)j * C, c, h);
      }
    } else {
#pragma unroll
      for (int j = 0; j < L; ++j) {
        h = PACKED && ((m.start | m.none) >> j & 1u) ? bb[j] : fma2(a[j], h, bb[j]);
        if (j < rows) Q::store(py + (long long)j * C, c, h);
        if (PACKED && (m.end >> j & 1u) && fin != nullptr)
          store_state(fin, seq_of(q, t0, j, m.end, m.end_seq), C, c, h);
      }
    }
  }
  if (!PACKED && fin != nullptr && rank == 0 && warp == 0) store_state(fin, b, C, c, carry);
  if (FAST) land_copies(bars + warp, waits->stuck[warp]);
  if (p.cs > 1) leave_cluster(waits, met, p.cs, rank, steps);
}

constexpr int REC_BW = REC_CKPT / REC_L;  // warps of a backward CTA: its tile starts from a kept state

template <typename T, bool FAST, bool PACKED, bool SERIES>
__device__ __forceinline__ void backward_body(const RecMaps &maps, SeqIn<T> x, SeqIn<T> u, SeqIn<T> v, const float *__restrict__ initial,
              const float *__restrict__ ckpt, SeqIn<T> dy, const float *__restrict__ dfin, T *__restrict__ dx,
              T *__restrict__ du, T *__restrict__ dv, float *__restrict__ dinit, float *__restrict__ part,
              const RecParams &p, const Rate &k) {
  using Q = Pair<T, FAST>;
  constexpr int L = REC_L, W = REC_BW, NT = 4, TILE = W * L;
  extern __shared__ __align__(128) unsigned char smem[];
  T *stage = reinterpret_cast<T *>(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (FAST ? rec_stage<T>(W, NT) : 0)), *met = bars + W;
  RecWaits *waits = reinterpret_cast<RecWaits *>(bars + 16);
  // P, H of each warp's rows, and what leaves them towards earlier rows
  float4(*agg)[W][32] = reinterpret_cast<float4(*)[W][32]>(reinterpret_cast<unsigned char *>(bars) + REC_BARRIERS);
  float2(*aggq)[W][32] = reinterpret_cast<float2(*)[W][32]>(agg + 2);
  float2(*keep)[32] = reinterpret_cast<float2(*)[32]>(aggq + 2) + uniform_warp() * L;  // a of this warp's rows
  float4 *far = reinterpret_cast<float4 *>(reinterpret_cast<float2(*)[32]>(aggq + 2) + W * L);  // [2][cs][32]
  const int lane = threadIdx.x & 31, warp = uniform_warp();
  const int rank = (int)(blockIdx.x % p.cs);
  const long long pair = blockIdx.x / p.cs;
  const int grp = (int)(pair % p.groups), b = (int)(pair / p.groups);
  const int C = p.q.C;
  const Chan c = Q::channels(grp, lane, C);
  const int tiles = ceil_div(p.q.T, TILE), steps = ceil_div(tiles, p.cs);
  T *mine = stage + warp * (NT * L * REC_GROUP);
  const int col = c.c0 - grp * REC_GROUP;  // of this lane in the staged rows
  auto start_copies = [&](int tile) {
    if (lane == 0 && look_at(waits->stuck[warp]) == 0) {
      const int t = tile * TILE + warp * L;
      mbar_arrive_expect_tx(bars + warp, NT * L * REC_GROUP * (uint32_t)sizeof(T));
#pragma unroll
      for (int n = 0; n < NT; ++n) rows_load(mine + n * L * REC_GROUP, &maps.m[n], grp * REC_GROUP, t, b, bars + warp);
    }
  };
  SeqList list = p.q;
  if (PACKED) {
    int *kept = reinterpret_cast<int *>(far + (p.cs > 1 ? 2 * p.cs * 32 : 0));
    keep_offsets(list, kept);
  }
  start_cta<W, FAST>(bars, waits, p, rank);
  if (FAST && steps > 0) start_copies((steps - 1) * p.cs + rank);
  if (PACKED && dinit != nullptr && rank == 0) empty_states<W>(p, warp, dfin, dinit, c);
  RowWalk walk;
  float2 carry = f2(0.f), ddecay = f2(0.f);
  if (!PACKED && dfin != nullptr) carry = load_state(dfin, b, C, c);
  RowMasks next_m{0u, 0u, 0u, -1, -1};
  if (PACKED && steps > 0) next_m = walk.masks<L>(list, ((steps - 1) * p.cs + rank) * TILE + warp * L);
  for (int it = steps - 1; it >= 0; --it) {
    const int n = steps - 1 - it, half = n & 1;
    const int tile = it * p.cs + rank, t0 = tile * TILE + warp * L;
    const int rows = p.q.T - t0;
    const RowMasks mk = next_m;
    const unsigned special = mk.start | mk.none;
    float2 h = f2(0.f);
    if (tile < tiles) h = load_state(ckpt, (long long)b * tiles + tile, C, c);
    typename Q::Raw rx[L];
    float2 t[L], i[L], g[L];
    {
      typename Q::Raw ru[L], rv[L], rg[L];
      if constexpr (FAST) {
        wait_copies(bars + warp, n & 1, p.polls, waits->stuck[warp]);
        if (!PACKED && rows < L) close_rows<T>(mine + L * REC_GROUP, rows, col);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          rx[j] = Q::P::load(mine + j * REC_GROUP + col);
          ru[j] = Q::P::load(mine + (L + j) * REC_GROUP + col);
          rv[j] = Q::P::load(mine + (2 * L + j) * REC_GROUP + col);
          rg[j] = Q::P::load(mine + (3 * L + j) * REC_GROUP + col);
        }
      } else {
        const T *px = x.row(b, t0), *pu = u.row(b, t0), *pv = v.row(b, t0), *pg = dy.row(b, t0);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          rx[j] = j < rows ? Q::load(px + j * x.rs, c) : Q::zero();
          ru[j] = j < rows ? Q::load(pu + j * u.rs, c) : Q::zero();
          if (!PACKED && j >= rows) ru[j] = Q::closed();
          rv[j] = j < rows ? Q::load(pv + j * v.rs, c) : Q::zero();
          rg[j] = j < rows ? Q::load(pg + j * dy.rs, c) : Q::zero();
        }
      }
#pragma unroll
      for (int j = 0; j < L; ++j) {
        if (PACKED && (mk.none >> j & 1u)) rx[j] = ru[j] = rv[j] = rg[j] = Q::zero();
        t[j] = root_sigmoid2(Q::get(ru[j]));
        i[j] = sigmoid2(Q::get(rv[j]));
        g[j] = Q::get(rg[j]);
      }
    }
    if constexpr (FAST) {
      if (!PACKED && rows < L) fence_proxy_async_smem();  // rows closed by plain stores
      __syncwarp();
      if (it > 0) start_copies(tile - p.cs);
    }
    if (PACKED && mk.end != 0u && dfin != nullptr) {
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (mk.end >> j & 1u)
          g[j] = add2(g[j], load_state(dfin, seq_of(list, t0, j, mk.end, mk.end_seq), C, c));
    }
    // what the rows do to a state going down (P, H), and what they pass to a gradient going up
    // (G = sum_j a[0] .. a[j] g[j], up to the first row that begins a sequence)
    float2 P = f2(1.f), H = f2(0.f), G = f2(0.f);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const float2 s = mul2(k.ks, mul2(t[j], t[j])), a = keep2<SERIES>(s);
      keep[j][lane] = a;
      float2 bb = mul2(beta2<SERIES>(t[j], s, k), mul2(i[j], Q::get(rx[j])));
      if (PACKED && (special >> j & 1u)) {
        if (mk.none >> j & 1u) bb = f2(0.f);
        else if (initial != nullptr)
          bb = fma2(a, load_state(initial, seq_of(list, t0, j, mk.start, mk.start_seq), C, c), bb);
        P = f2(-1.f);
        H = bb;
      } else {
        P = join<PACKED>(P, a);
        H = fma2(a, H, bb);
        if (!PACKED || !cut(P)) G = fma2(P, g[j], G);
      }
    }
#pragma unroll
    for (int j = 0; j < L; ++j) {
      forget(t[j]);
      forget(i[j]);
    }
    agg[half][warp][lane] = make_float4(P.x, P.y, H.x, H.y);
    aggq[half][warp][lane] = G;
    __syncthreads();
    if (PACKED && it > 0) next_m = walk.masks<L>(list, t0 - p.cs * TILE);
    float2 q = carry;
    if (p.cs > 1) {
      float4 *there = far + (half * p.cs + rank) * 32 + lane;
      const bool part = look_at(waits->give_up) > n;
      if (warp < p.cs) {
        float2 TP = f2(1.f), TG = f2(0.f);
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
          const float4 e = agg[half][w][lane];
          const float2 P2 = make_float2(e.x, e.y);
          TG = apply<PACKED>(P2, aggq[half][w][lane], TG);
          TP = join<PACKED>(TP, P2);
        }
        if (part) {
          for (int peer = warp; peer < p.cs; peer += W)
            store_peer(there, met + half, peer, make_float4(TP.x, TP.y, TG.x, TG.y));
          if (threadIdx.x == 0) mbar_arrive_expect_tx(met + half, p.cs * 512);
        }
      }
      if (part) wait_peers(met + half, n, p.polls, waits->give_up);
      for (int w = p.cs - 1; w >= 0; --w) {
        if (w == rank) q = carry;
        const float4 e = far[(half * p.cs + w) * 32 + lane];
        carry = apply<PACKED>(make_float2(e.x, e.y), make_float2(e.z, e.w), carry);
      }
    }
    float2 in = q;
#pragma unroll
    for (int w = W - 1; w >= 0; --w) {
      if (w == warp) {
        in = q;
        if (p.cs > 1) break;
      }
      const float4 e = agg[half][w][lane];
      q = apply<PACKED>(make_float2(e.x, e.y), aggq[half][w][lane], q);
    }
    if (p.cs == 1) carry = q;
    q = in;
    for (int w = 0; w < warp; ++w) {
      const float4 e = agg[half][w][lane];
      h = apply<PACKED>(make_float2(e.x, e.y), make_float2(e.z, e.w), h);
    }
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
      g[j] = add2(g[j], q);
      q = mul2(keep[j][lane], g[j]);
      if (PACKED && (special >> j & 1u)) {
        if ((mk.start >> j & 1u) && dinit != nullptr)
          store_state(dinit, seq_of(list, t0, j, mk.start, mk.start_seq), C, c, q);
        q = f2(0.f);
      }
    }
    const long long at = ((long long)b * p.q.T + t0) * C;
    T *px = dx + at, *pu = du + at, *pv = dv + at;
    float2 sum = f2(0.f);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const float2 a = keep[j][lane], r = mul2(t[j], t[j]), s = mul2(k.ks, r);
      const float2 beta = beta2<SERIES>(t[j], s, k), rho = rho2<SERIES>(t[j], s, k);
      const float2 xv = Q::get(rx[j]), ix = mul2(i[j], xv);
      if (PACKED && (special >> j & 1u)) {
        h = f2(0.f);
        if ((mk.start >> j & 1u) && initial != nullptr)
          h = load_state(initial, seq_of(list, t0, j, mk.start, mk.start_seq), C, c);
      }
      float2 ddx = mul2(g[j], mul2(beta, i[j]));
      float2 ddv = mul2(mul2(ddx, xv), one_minus2(i[j]));
      float2 dzz = mul2(mul2(g[j], a), fma2(mul2(a, rho), ix, mul2(s, h)));
      float2 ddu = mul2(dzz, one_minus2(r));
      if (PACKED && (mk.none >> j & 1u)) ddx = ddv = dzz = ddu = f2(0.f);  // whatever the channel's decay
      sum = add2(sum, dzz);
      h = fma2(a, h, mul2(beta, ix));
      if (j < rows) {
        Q::store(px + (long long)j * C, c, ddx);
        Q::store(pu + (long long)j * C, c, ddu);
        Q::store(pv + (long long)j * C, c, ddv);
      }
    }
    ddecay = add2(ddecay, sum);
  }
  if (!PACKED && dinit != nullptr && rank == 0 && warp == 0) store_state(dinit, b, C, c, carry);
  if (FAST) land_copies(bars + warp, waits->stuck[warp]);
  // this CTA's part of ddecay: the warps' sums in order
  __syncthreads();
  aggq[0][warp][lane] = ddecay;
  __syncthreads();
  if (warp == 0) {
    float2 s = aggq[0][0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s = add2(s, aggq[0][w][lane]);
    store_state(part, (long long)b * p.cs + rank, C, c, s);
  }
  if (p.cs > 1) leave_cluster(waits, met, p.cs, rank, steps);
}

__device__ __forceinline__ Rate rate_of(const float *decay, float scale, const Chan &c) {
  const float2 k = make_float2(scale * softplus(decay[c.c0]), scale * softplus(decay[c.c1]));
  return Rate{make_float2(-k.x, -k.y), make_float2(sqrtf(2.f * k.x), sqrtf(2.f * k.y))};
}
template <typename T, bool FAST> __device__ __forceinline__ Rate cta_rate(const float *decay, const RecParams &p) {
  const int grp = (int)(blockIdx.x / p.cs % p.groups);
  return rate_of(decay, p.scale, Pair<T, FAST>::channels(grp, threadIdx.x & 31, p.q.C));
}

// CTAs per SM that the registers are cut for.  (Eight warps with two CTAs per SM and 128 registers took 160 us
// where three took 133 on 32768 fp32 rows of 1152 channels: clusters of 16 then leave SMs of a GPC unused.)
constexpr int rec_forward_ctas(int W) { return W == 4 ? 8 : 3; }
constexpr int REC_BACKWARD_CTAS = 4;

template <typename T, int W, bool FAST, bool PACKED>
__global__ void __launch_bounds__(W * 32, rec_forward_ctas(W))
recurrence_forward_kernel(const __grid_constant__ RecMaps maps, SeqIn<T> x, SeqIn<T> u, SeqIn<T> v,
                          const float *__restrict__ decay, const float *__restrict__ initial, T *__restrict__ y,
                          float *__restrict__ fin, float *__restrict__ ckpt, RecParams p) {
  const Rate k = cta_rate<T, FAST>(decay, p);
  // the same in every warp of the CTA: they have its channels in common
  if (__all_sync(0xffffffffu, k.ks.x >= -REC_SERIES && k.ks.y >= -REC_SERIES))
    forward_body<T, W, FAST, PACKED, true>(maps, x, u, v, initial, y, fin, ckpt, p, k);
  else
    forward_body<T, W, FAST, PACKED, false>(maps, x, u, v, initial, y, fin, ckpt, p, k);
}

template <typename T, bool FAST, bool PACKED>
__global__ void __launch_bounds__(REC_BW * 32, REC_BACKWARD_CTAS)
recurrence_backward_kernel(const __grid_constant__ RecMaps maps, SeqIn<T> x, SeqIn<T> u, SeqIn<T> v, const float *__restrict__ decay,
                           const float *__restrict__ initial, const float *__restrict__ ckpt, SeqIn<T> dy,
                           const float *__restrict__ dfin, T *__restrict__ dx, T *__restrict__ du, T *__restrict__ dv,
                           float *__restrict__ dinit, float *__restrict__ part, RecParams p) {
  const Rate k = cta_rate<T, FAST>(decay, p);
  if (__all_sync(0xffffffffu, k.ks.x >= -REC_SERIES && k.ks.y >= -REC_SERIES))
    backward_body<T, FAST, PACKED, true>(maps, x, u, v, initial, ckpt, dy, dfin, dx, du, dv, dinit, part, p, k);
  else
    backward_body<T, FAST, PACKED, false>(maps, x, u, v, initial, ckpt, dy, dfin, dx, du, dv, dinit, part, p, k);
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
  const int C = p.q.C;
  const Chan c = Q::channels(grp, lane, C);
  const typename Q::Raw rx = Q::load(x + b * xs, c), ru = Q::load(u + b * us, c), rv = Q::load(v + b * vs, c);
  const float2 h0 = load_state(state, b, C, c);
  const Rate k = rate_of(decay, p.scale, c);
  const float2 t = root_sigmoid2(Q::get(ru)), sz = mul2(k.ks, mul2(t, t));
  const float2 bb = mul2(beta2<false>(t, sz, k), mul2(sigmoid2(Q::get(rv)), Q::get(rx)));
  const float2 h = fma2(keep2<false>(sz), h0, bb);
  __syncwarp();  // lanes that share a channel have all read its state
  store_state(state, b, C, c, h);
  Q::store(y + b * C, c, h);
}

// ---- host --------------------------------------------------------------------------------------

// A kernel's CTA, and what is known about its time: a tile takes `tile` microseconds of an SM's throughput, and
// `chain` where the SM has nothing else to do (its loads, gates, folds and exchanges follow one another).
struct RecShape {
  int W, stage, ctas;
  bool backward, packed;
  float tile, chain;
  int smem(int cs) const { return rec_smem(W, stage, backward, packed, cs); }
};

// CTAs of a cluster along T, and the time that goes with it in microseconds, by a model: n CTAs of an SM take
// (tile n) and (chain) per tile, the larger nearly alone; CTAs beyond those that fit follow them; a start
// is worth two tiles.  It is for choosing alone: its times are near for many channels (475 us and 432 measured) and
// too short for few (packed list below: 50 and 76; 32771 fp32 rows of 1152: 98 and 135), since it knows neither
// sequence borders nor the wider type nor the eight-warp packed kernel's spills (440 bytes loaded).  Measured
// against all sizes: one packed list of 8191 rows of 2560 channels in bf16, forward, eight warps, clusters of
// 4 / 6 / 8 / 10 / 12 / 16: 115 / 90 / 86 / 74 / 104 / 96 us (it takes 10); 8 x 8192 rows of 4096, backward, 1 / 2 / 4 / 8:
// 971 / 893 / 944 / 985 us (it takes 2); 4 x 2048 rows of 2048, backward, 2 / 4 / 6 / 8 / 10: 92 / 82 / 86 / 84 / 94 (it
// takes 8).  Odd sizes and 14 leave SMs of a GPC without work and are not in the choice.
struct RecChoice {
  int cs;
  float us;
};
inline RecChoice rec_cluster(const dwconv_b200_sequence &s, const RecShape &r) {
  static const int sizes[] = {1, 2, 4, 6, 8, 10, 12, 16};
  const int sms = 148, tiles = ceil_div(s.T, r.W * REC_L);
  const long long pairs = (long long)ceil_div(s.C, REC_GROUP) * s.B;
  RecChoice best{1, 0.f};
  for (int cs : sizes) {
    if (cs > 1 && cs > tiles) break;
    const int fit = 227 * 1024 / (r.smem(cs) + 1024), slots = fit < r.ctas ? fit : r.ctas;
    auto time = [&](float n) {
      const float a = r.tile * n, b = r.chain;
      return sqrtf(sqrtf(a * a * a * a + b * b * b * b));
    };
    const float n = (float)(pairs * cs) / sms, full = floorf(n / slots), rest = ceilf(n - full * slots);
    const float us = (ceil_div(tiles, cs) + 2) * (full * time((float)slots) + (rest > 0.f ? time(rest) : 0.f));
    if (cs == 1 || us < best.us) best = RecChoice{cs, us};
  }
  return best;
}

std::atomic<int> g_expire{0};  // dwconv_b200_debug_expire
constexpr unsigned REC_SHORT_POLLS = 64;  // some milliseconds

inline RecParams rec_params(const dwconv_b200_sequence &s, float scale, int cs) {
  RecParams p;
  const int expire = g_expire.load(std::memory_order_relaxed);
  p.polls = expire == 0 ? ROWS_WAIT_LIMIT : (expire == 1 ? 0 : REC_SHORT_POLLS);
  p.leaver = expire == 2 ? cs - 1 : -1;
  p.q = seq_list(s);
  p.B = s.B;
  p.groups = ceil_div(s.C, REC_GROUP);
  p.cs = cs;
  p.scale = scale;
  return p;
}

// Launches `kernel` in clusters of p.cs CTAs.  The attributes that this takes are set once per kernel and
// device.
template <typename... K, typename... A>
void rec_launch(void (*kernel)(K...), std::atomic<unsigned long long> &ready, const RecParams &p, const RecShape &r,
                cudaStream_t st, A... args) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return;
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, r.smem(REC_MAX_CLUSTER)) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return;  // the caller finds the error
    ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)p.groups * p.B * p.cs));
  cfg.blockDim = dim3(r.W * 32);
  cfg.dynamicSmemBytes = r.smem(p.cs);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cs > 1 ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, kernel, args...);
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

// One operand as the copy engine sees it; false where it cannot.
template <typename T> bool rows_map(CUtensorMap *map, const dwconv_b200_rows &r, const dwconv_b200_sequence &s) {
  constexpr int E = 16 / (int)sizeof(T);
  // the stride of an extent of one is never used: any valid one will do
  const long long rs = s.T > 1 ? r.row_stride : E, bs = s.B > 1 ? r.batch_stride : E;
  if (!aligned_to(r.data, 16) || rs <= 0 || bs <= 0 || rs % E != 0 || bs % E != 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)s.C, (cuuint64_t)s.T, (cuuint64_t)s.B};
  const cuuint64_t strides[2] = {(cuuint64_t)rs * sizeof(T), (cuuint64_t)bs * sizeof(T)};
  const cuuint32_t box[3] = {(cuuint32_t)REC_GROUP, (cuuint32_t)REC_L, 1u};
  return encode_tensor_map<T>(map, static_cast<const T *>(r.data), 3, dims, strides, box);
}
template <typename T> bool rec_maps(const RecArgs &a, RecMaps &maps) {
  if (a.s->T == 0 || a.s->C % 2 != 0) return false;
  const void *ptrs[] = {a.y, a.dx, a.du, a.dv};
  for (const void *q : ptrs)
    if (q != nullptr && !aligned_to(q, 2 * sizeof(T))) return false;
  return rows_map<T>(&maps.m[0], *a.x, *a.s) && rows_map<T>(&maps.m[1], *a.u, *a.s) &&
         rows_map<T>(&maps.m[2], *a.v, *a.s) && (a.dy == nullptr || rows_map<T>(&maps.m[3], *a.dy, *a.s));
}

template <typename T, int W, bool FAST, bool PACKED> RecShape forward_shape() {
  return RecShape{W, FAST ? rec_stage<T>(W, 3) : 0, rec_forward_ctas(W), false, PACKED, W * 0.125f, W == 4 ? 2.3f : 2.6f};
}
template <typename T, int W, bool FAST, bool PACKED>
void launch_forward(const RecArgs &a, const RecMaps &maps, int cs, cudaStream_t st) {
  static std::atomic<unsigned long long> ready{0};
  const RecParams p = rec_params(*a.s, a.scale, cs);
  rec_launch(recurrence_forward_kernel<T, W, FAST, PACKED>, ready, p, forward_shape<T, W, FAST, PACKED>(), st, maps,
             seq_in<T>(*a.x), seq_in<T>(*a.u), seq_in<T>(*a.v), a.decay, a.initial, static_cast<T *>(a.y), a.fin, a.ckpt,
             p);
}
template <typename T, bool FAST, bool PACKED>
int launch_backward(const RecArgs &a, const RecMaps &maps, cudaStream_t st) {
  static std::atomic<unsigned long long> ready{0};
  const RecShape r{REC_BW, FAST ? rec_stage<T>(REC_BW, 4) : 0, REC_BACKWARD_CTAS, true, PACKED, 1.f, 2.4f};
  const RecParams p = rec_params(*a.s, a.scale, rec_cluster(*a.s, r).cs);
  rec_launch(recurrence_backward_kernel<T, FAST, PACKED>, ready, p, r, st, maps, seq_in<T>(*a.x), seq_in<T>(*a.u),
             seq_in<T>(*a.v), a.decay, a.initial, a.ckpt_in, seq_in<T>(*a.dy), a.dfin, static_cast<T *>(a.dx),
             static_cast<T *>(a.du), static_cast<T *>(a.dv), a.dinit, a.part, p);
  return p.cs;
}

// CTAs of four warps have the cheapest barriers and pack best; those of eight take twice the rows between two
// exchanges, which counts where there are few of them.  8 x 8192 rows of 4096 channels in bf16: 432 us with
// four, 447 with eight; one sequence of 32771 fp32 rows of 1152: 158 and 135; the packed list above: 92 and 74.
template <typename T, bool FAST, bool PACKED> void forward_v(const RecArgs &a, const RecMaps &maps, cudaStream_t st) {
  const RecChoice four = rec_cluster(*a.s, forward_shape<T, 4, FAST, PACKED>());
  const RecChoice eight = rec_cluster(*a.s, forward_shape<T, 8, FAST, PACKED>());
  if (four.us <= eight.us) launch_forward<T, 4, FAST, PACKED>(a, maps, four.cs, st);
  else launch_forward<T, 8, FAST, PACKED>(a, maps, eight.cs, st);
}
template <typename T> void forward_t(const RecArgs &a, cudaStream_t st) {
  const bool packed = a.s->offsets != nullptr;
  RecMaps maps{};
  if (rec_maps<T>(a, maps)) packed ? forward_v<T, true, true>(a, maps, st) : forward_v<T, true, false>(a, maps, st);
  else packed ? forward_v<T, false, true>(a, maps, st) : forward_v<T, false, false>(a, maps, st);
}
// Returns the CTAs of a cluster: each left a part of the decay's gradient.
template <typename T> int backward_t(const RecArgs &a, cudaStream_t st) {
  const bool packed = a.s->offsets != nullptr;
  RecMaps maps{};
  if (rec_maps<T>(a, maps))
    return packed ? launch_backward<T, true, true>(a, maps, st) : launch_backward<T, true, false>(a, maps, st);
  return packed ? launch_backward<T, false, true>(a, maps, st) : launch_backward<T, false, false>(a, maps, st);
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

// Reads and clears this translation unit's error flag (bit 3).
int seq_take_error() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_seq_error_flag, sizeof(int)) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  if (v != 0) {
    const int zero = 0;
    (void)cudaMemcpyToSymbol(g_seq_error_flag, &zero, sizeof(int));
  }
  return v;
}

}  // namespace dwb

using namespace dwb;

extern "C" {

int dwconv_b200_debug_expire(int how) { return g_expire.exchange(how == 1 || how == 2 ? how : 0); }

size_t dwconv_b200_recurrence_checkpoint_bytes(const dwconv_b200_sequence *seq) {
  if (check_recurrence(DWCONV_B200_F32, seq) != DWCONV_B200_OK) return 0;
  const size_t n = (size_t)seq->B * ceil_div(seq->T, REC_CKPT) * seq->C * sizeof(float);
  return (n + 15) / 16 * 16 + 16;
}

size_t dwconv_b200_recurrence_workspace_bytes(const dwconv_b200_sequence *seq) {
  if (check_recurrence(DWCONV_B200_F32, seq) != DWCONV_B200_OK) return 0;
  const size_t n = (size_t)seq->B * REC_MAX_CLUSTER * seq->C * sizeof(float);
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
  int cs = 1;
  switch (dtype) {
    case DWCONV_B200_F32: cs = backward_t<float>(a, st); break;
    case DWCONV_B200_F16: cs = backward_t<__half>(a, st); break;
    default: cs = backward_t<__nv_bfloat16>(a, st); break;
  }
  e = api_launch_status();
  if (e) return e;
  launch_column_sum(a.part, (long long)seq->B * cs, seq->C,
                    ColumnSumOut{ddecay, nullptr, DWCONV_B200_F32, seq->C, 1, decay}, st);
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
  RecParams p{};
  p.q = seq_list(s);
  p.B = B;
  p.groups = ceil_div(C, REC_GROUP);
  p.cs = 1;
  p.scale = scale;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case DWCONV_B200_F32: step_t<float>(x, x_stride, u, u_stride, v, v_stride, decay, state, y, p, st); break;
    case DWCONV_B200_F16: step_t<__half>(x, x_stride, u, u_stride, v, v_stride, decay, state, y, p, st); break;
    default: step_t<__nv_bfloat16>(x, x_stride, u, u_stride, v, v_stride, decay, state, y, p, st); break;
  }
  return api_launch_status();
}

}  // extern "C"
