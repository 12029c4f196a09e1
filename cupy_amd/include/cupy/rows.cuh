// Helpers of the hand-written row kernels (norms, log probabilities, table
// gradients): the type sums are held in, partial vectors at the end of a row,
// and all-reduces over the lanes that share a row.
#pragma once
#include <cupy/carray.cuh>

namespace cupy {

// Statistics are held in 32 bits for float16 and float32, in 64 for float64.
template <typename T> struct acc_of { typedef float type; };
template <> struct acc_of<double> { typedef double type; };

template <typename A> struct bits_of { typedef unsigned int type; };
template <> struct bits_of<double> { typedef unsigned long long type; };

_CUPY_DEV float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
_CUPY_DEV double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }
_CUPY_DEV float sqrt_(float a) { return __builtin_sqrtf(a); }
_CUPY_DEV double sqrt_(double a) { return __builtin_sqrt(a); }
_CUPY_DEV float rint_(float a) { return __builtin_rintf(a); }
_CUPY_DEV double rint_(double a) { return __builtin_rint(a); }
_CUPY_DEV float abs_(float a) { return __builtin_fabsf(a); }
_CUPY_DEV double abs_(double a) { return __builtin_fabs(a); }

// |a| as an integer that orders like |a|, with NaN above infinity: a maximum
// over these keeps a NaN, which the floating-point maximum drops.
_CUPY_DEV unsigned int abs_bits(float a) { return __builtin_bit_cast(unsigned int, a) & 0x7fffffffu; }
_CUPY_DEV unsigned long long abs_bits(double a) {
  return __builtin_bit_cast(unsigned long long, a) & 0x7fffffffffffffffull;
}
_CUPY_DEV float from_bits(unsigned int b) { return __builtin_bit_cast(float, b); }
_CUPY_DEV double from_bits(unsigned long long b) { return __builtin_bit_cast(double, b); }

// The first `have` of N elements (have >= N: one vector access), zeros behind them.
template <typename T, int N, bool kStream = false>
_CUPY_DEV Vec<T, N> load_part(const T* p, int have) {
  if (have >= N) return load_vec<T, N, kStream>(p);
  Vec<T, N> r;
#pragma unroll
  for (int e = 0; e < N; ++e) r.v[e] = e < have ? p[e] : static_cast<T>(0.0f);
  return r;
}
template <typename T, int N, bool kStream = false>
_CUPY_DEV void store_part(T* p, const Vec<T, N>& x, int have) {
  if (have >= N) {
    store_vec<T, N, kStream>(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) if (e < have) p[e] = x.v[e];
  }
}

// The kItems vectors of a row that one of kLanes lanes works on.  All of them are
// loaded without a branch between the requests: a vector that would hang over
// the end of the row is moved back to end with it, and one wholly behind it as
// well.  What a moved vector shares with its neighbours is theirs: it is left
// out of sums (`owns`), and stored twice with the same values.
// kTiny: rows shorter than a vector, loaded and stored by elements.
template <int kItems, int kLanes, int kVec, bool kTiny>
struct RowShare {
  int width;
  int at[kItems];       // first column, as loaded
  int skip[kItems];     // elements of it that are not this lane's
  _CUPY_DEV RowShare(int lane, int w) : width(w) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int c = (lane + k * kLanes) * kVec;
      at[k] = kTiny ? 0 : c + kVec <= w ? c : w - kVec;
      const int s = c - at[k];
      skip[k] = s < kVec ? s : kVec;
    }
  }
  _CUPY_DEV bool owns(int k, int e) const { return e >= skip[k] && (!kTiny || e < width); }
  _CUPY_DEV bool any(int k) const { return skip[k] < kVec; }
  template <bool kStream = false, typename T>
  _CUPY_DEV void load(Vec<T, kVec> (&v)[kItems], const T* row) const {
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      v[k] = kTiny ? load_part<T, kVec>(row, width) : load_vec<T, kVec, kStream>(row + at[k]);
  }
  template <bool kStream, typename T>
  _CUPY_DEV void store(int k, T* row, const Vec<T, kVec>& v) const {
    if (kTiny) store_part<T, kVec>(row, v, width);
    else store_vec<T, kVec, kStream>(row + at[k], v);
  }
};

constexpr int _ceil_pow2(int n, int p = 1) { return p >= n ? p : _ceil_pow2(n, 2 * p); }

// All-reduce over the kLanes lanes of a row: a group inside a wave (a power of
// two), or the whole workgroup of kLanes == kBlock threads, any number of
// waves, through `lds` (a value per wave).  A value of zeros has to be the
// identity of `op`.  A workgroup that calls this repeatedly alternates between
// two such arrays: one barrier per call is enough then, because whoever writes
// an array for the second time has passed the barrier of the call in between.
template <int kLanes, int kBlock, typename T, typename Op>
_CUPY_DEV T row_allreduce(T v, Op op, T* lds) {
  if (kLanes <= 64) return group_allreduce<(kLanes <= 64 ? kLanes : 64)>(v, op);
  constexpr int kWaves = kBlock / 64 > 0 ? kBlock / 64 : 1;
  constexpr int kGroup = _ceil_pow2(kWaves);
  v = group_allreduce<64>(v, op);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  const int from = threadIdx.x & (kGroup - 1);
  T w = lds[from < kWaves ? from : 0];
  if (from >= kWaves) w = T();
  return group_allreduce<kGroup>(w, op);
}

}  // namespace cupy
