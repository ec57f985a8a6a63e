// Shared pieces of the sequence operators (causal depthwise conv1d, gated linear recurrence, layer
// norm): rows of channels that lie side by side, loaded V channels at a time and worked on in fp32.
#pragma once

#include "api_checks.cuh"
#include "common.cuh"

namespace dwb {

// One operand of a sequence operator: element (b, t, c) at data[b * bs + t * rs + c].
template <typename T> struct SeqIn {
  const T *p;
  long long bs, rs;
  __device__ __forceinline__ const T *row(int b, long long t) const { return p + b * bs + t * rs; }
};

// One element as fp32.  Plain loads throughout these kernels: many stand behind a bounds or a null
// check, and the load intrinsics of some types are assembly that the compiler may execute before it.
template <typename T> __device__ __forceinline__ float read(const T *p) { return Elem<T>::to_acc(*p); }

// V adjacent elements as they lie in memory, moved by one load or store.
template <int BYTES> struct RawVec;
template <> struct RawVec<2> { using type = unsigned short; };
template <> struct RawVec<4> { using type = uint32_t; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<16> { using type = uint4; };

template <typename T, int V> struct Pack {
  using Raw = typename RawVec<V * (int)sizeof(T)>::type;
  static __device__ __forceinline__ Raw load(const T *p) { return *reinterpret_cast<const Raw *>(p); }
  static __device__ __forceinline__ void store(T *p, const Raw &r) { *reinterpret_cast<Raw *>(p) = r; }
  static __device__ __forceinline__ Raw zero() {
    Raw r;
    memset(&r, 0, sizeof(r));
    return r;
  }
  static __device__ __forceinline__ void unpack(const Raw &r, float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
      memcpy(f, &r, sizeof(r));
    } else if constexpr (V == 1) {
      f[0] = Pack16<T>::from_bits(r);
    } else {
      uint32_t w[V / 2];
      memcpy(w, &r, sizeof(r));
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 q = Pack16<T>::unpack(w[i]);
        f[2 * i] = q.x;
        f[2 * i + 1] = q.y;
      }
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[V]) {
    Raw r;
    if constexpr (sizeof(T) == 4) {
      memcpy(&r, f, sizeof(r));
    } else if constexpr (V == 1) {
      r = Pack16<T>::to_bits(f[0]);
    } else {
      uint32_t w[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = Pack16<T>::pack(f[2 * i], f[2 * i + 1]);
      memcpy(&r, w, sizeof(r));
    }
    return r;
  }
};

// ---- channels of a lane ------------------------------------------------------------------------

// Arithmetic on pairs of channels: one instruction for two fp32 operations.
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 one_minus2(float2 v) { return fma2(v, f2(-1.f), f2(1.f)); }

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

// 1 + exp(-v)
__device__ __forceinline__ float2 one_plus_exp2(float2 v) {
  const float2 e = mul2(v, f2(-LOG2E));
  return add2(make_float2(ex2f(e.x), ex2f(e.y)), f2(1.f));
}
// sigmoid; an overflowing exponential gives 0
__device__ __forceinline__ float2 sigmoid2(float2 v) {
  const float2 s = one_plus_exp2(v);
  return make_float2(rcpf(s.x), rcpf(s.y));
}

// H pairs of channels per lane.  VEC: 2 H adjacent ones, one load; otherwise (odd C, odd strides; H = 1)
// channels c and d = c + 32, one load each.  Lanes beyond the last channel work on the last ones too, and
// store the same values to the same places: no access needs a test.
template <typename T, int H, bool VEC> struct Lanes;
template <typename T, int H> struct Lanes<T, H, true> {
  static constexpr int GROUP = 64 * H;  // channels of a warp
  using P = Pack<T, 2 * H>;
  using Raw = typename P::Raw;
  int c;
  __device__ __forceinline__ Lanes(int group, int lane, int C) : c(min(group * GROUP + 2 * H * lane, C - 2 * H)) {}
  __device__ __forceinline__ int channel(int i) const { return c + i; }
  __device__ __forceinline__ Raw load(const T *row) const { return P::load(row + c); }
  __device__ __forceinline__ void store(T *row, const float2 (&v)[H]) const {
    float f[2 * H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      f[2 * h] = v[h].x;
      f[2 * h + 1] = v[h].y;
    }
    P::store(row + c, P::pack(f));
  }
  static __device__ __forceinline__ Raw zero() { return P::zero(); }
  static __device__ __forceinline__ void get(const Raw &r, float2 (&v)[H]) {
    float f[2 * H];
    P::unpack(r, f);
#pragma unroll
    for (int h = 0; h < H; ++h) v[h] = make_float2(f[2 * h], f[2 * h + 1]);
  }
};
template <typename T> struct Lanes<T, 1, false> {
  static constexpr int GROUP = 64;
  struct Raw { T a, b; };
  int c, d;
  __device__ __forceinline__ Lanes(int group, int lane, int C)
      : c(min(group * GROUP + lane, C - 1)), d(min(group * GROUP + lane + 32, C - 1)) {}
  __device__ __forceinline__ int channel(int i) const { return i ? d : c; }
  __device__ __forceinline__ Raw load(const T *row) const { return Raw{row[c], row[d]}; }
  __device__ __forceinline__ void store(T *row, const float2 (&v)[1]) const {
    row[c] = Elem<T>::from_acc(v[0].x);
    row[d] = Elem<T>::from_acc(v[0].y);
  }
  static __device__ __forceinline__ Raw zero() { return Raw{Elem<T>::from_acc(0.f), Elem<T>::from_acc(0.f)}; }
  static __device__ __forceinline__ void get(const Raw &r, float2 (&v)[1]) {
    v[0] = make_float2(Elem<T>::to_acc(r.a), Elem<T>::to_acc(r.b));
  }
};

// ---- packed sequences --------------------------------------------------------------------------

// The list of packed sequences, or (offsets null) one sequence per batch element.
struct SeqList {
  int T, C;
  const int *offsets;  // S + 1 entries, or null
  int S;               // sequences (with offsets), else the batch size
};

// Entry j as a row number inside [0, T], whatever the caller wrote there.
__device__ __forceinline__ int seq_bound(const SeqList &q, int j) {
  const int v = q.offsets[j];
  return v < 0 ? 0 : (v > q.T ? q.T : v);
}

// Where row t lies.
struct SeqSpan {
  int seq;      // its sequence, -1 for a row of none
  int begin;    // first row of the sequence (of the run of rows of none)
  int next;     // first row behind it that belongs to something else, > t
};

// Last j with offsets[j] <= t, by bisection; every value read is clamped, so a list that is not
// ascending gives some sequence, never an access outside the tensors.
__device__ __forceinline__ SeqSpan seq_locate(const SeqList &q, int t) {
  int lo = 0, hi = q.S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (seq_bound(q, mid) <= t) lo = mid;
    else hi = mid;
  }
  const int s = seq_bound(q, lo), e = seq_bound(q, lo + 1);
  SeqSpan r;
  if (s <= t && t < e) {
    r.seq = lo; r.begin = s; r.next = e;
  } else if (s > t) {  // before the first sequence
    r.seq = -1; r.begin = 0; r.next = s;
  } else {  // behind the last one
    r.seq = -1; r.begin = e <= t ? e : t; r.next = q.T;
  }
  return r;
}

// ---- column sums -------------------------------------------------------------------------------

// Where the sum of one column of a [parts][M] table of fp32 partial sums goes: the first `split`
// columns to `first`, the rest to `second`; column m = k * C + c of the first part lands at
// c * K + k (the filter layout), K = 1 keeps the order.
struct ColumnSumOut {
  void *first, *second;
  int dtype;
  int C, K;             // split = C * K
  const float *decay;   // non-null: the sum of column c times sigmoid(decay[c]) / softplus(decay[c])
};

constexpr int COLSUM_LANES = 32, COLSUM_WARPS = 32;

__device__ __forceinline__ void store_as(void *p, long long i, float v, int dtype) {
  if (dtype == DWCONV_B200_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == DWCONV_B200_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// Every column is added in the same order on every run: warp w takes parts w, w + 32, ..., four at a time.
static __global__ void __launch_bounds__(COLSUM_LANES *COLSUM_WARPS)
column_sum_kernel(const float *__restrict__ part, long long parts, int M, ColumnSumOut out) {
  __shared__ float s[COLSUM_WARPS][COLSUM_LANES];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int m = blockIdx.x * COLSUM_LANES + lane;
  float acc = 0.f;
  pdl_wait();  // the kernel that left the parts has finished
  if (m < M)
    for (long long p = w; p < parts; p += 4 * COLSUM_WARPS) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long q = p + i * COLSUM_WARPS;
        v[i] = q < parts ? part[q * M + m] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) acc += v[i];
    }
  s[w][lane] = acc;
  __syncthreads();
  // eight warps add four of the sums each, one warp theirs
  if (w < 8) {
    acc = s[w][lane];
#pragma unroll
    for (int i = 1; i < 4; ++i) acc += s[w + 8 * i][lane];
  }
  __syncthreads();
  if (w < 8) s[w][lane] = acc;
  __syncthreads();
  if (w != 0 || m >= M) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += s[i][lane];
  const int split = out.C * out.K;
  if (out.decay != nullptr && m < split) {
    const float d = out.decay[m];
    // the quotient tends to 1 for far negative values, where both vanish
    v *= d < -80.f ? 1.f : 1.f / ((1.f + expf(-d)) * (d > 20.f ? d : log1pf(expf(d))));
  }
  if (m < split) {
    const int k = m / out.C, c = m - k * out.C;
    if (out.first) store_as(out.first, (long long)c * out.K + k, v, out.dtype);
  } else if (out.second) {
    store_as(out.second, m - split, v, out.dtype);
  }
}

// Launched so that its start-up runs under the end of the kernel that leaves the parts.
inline void launch_column_sum(const float *part, long long parts, int M, const ColumnSumOut &out, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ceil_div(M, COLSUM_LANES));
  cfg.blockDim = dim3(COLSUM_LANES * COLSUM_WARPS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  (void)cudaLaunchKernelEx(&cfg, column_sum_kernel, part, parts, M, out);
}

// ---- host checks -------------------------------------------------------------------------------

inline bool seq_dtype_ok(int dtype) {
  return dtype == DWCONV_B200_F32 || dtype == DWCONV_B200_F16 || dtype == DWCONV_B200_BF16;
}

inline int check_sequence(const dwconv_b200_sequence *s) {
  if (s == nullptr || s->B <= 0 || s->C <= 0 || s->T < 0 || s->S < 0) return DWCONV_B200_BAD_ARGUMENT;
  if (s->offsets != nullptr && (s->B != 1 || s->S < 1 || !aligned_to(s->offsets, 4)))
    return DWCONV_B200_BAD_ARGUMENT;
  // row numbers are 32-bit (with room for a tile behind the last); offsets into tensors 64-bit
  if (s->T > (1 << 30) || s->C > (1 << 26) || s->B > (1 << 26) || s->S > (1 << 26))
    return DWCONV_B200_TOO_LARGE;
  return DWCONV_B200_OK;
}

inline int check_rows(const dwconv_b200_rows *r, size_t es) {
  if (r == nullptr || r->data == nullptr) return DWCONV_B200_BAD_ARGUMENT;
  return aligned_to(r->data, es) ? DWCONV_B200_OK : DWCONV_B200_MISALIGNED;
}

// Whether rows can be moved `v` elements (v * es bytes) at a time.
inline bool rows_vector(const dwconv_b200_rows &r, int v, size_t es) {
  return aligned_to(r.data, v * es) && r.batch_stride % v == 0 && r.row_stride % v == 0;
}

template <typename T> inline SeqIn<T> seq_in(const dwconv_b200_rows &r) {
  return SeqIn<T>{static_cast<const T *>(r.data), r.batch_stride, r.row_stride};
}

inline SeqList seq_list(const dwconv_b200_sequence &s) {
  return SeqList{s.T, s.C, static_cast<const int *>(s.offsets), s.offsets ? s.S : s.B};
}

}  // namespace dwb
