"""Root-mean-square norm of rows: with the addition of a residual, with an
output in 8 bits, and its gradient.

With ``h = x + residual`` (``h = x`` without one) a row of ``width`` elements
becomes ``y = h * r * weight``, ``r = 1 / sqrt(mean(h * h) + eps)``.  A row is
read once: a group of lanes holds it in registers (packed, as it is stored),
reduces, and writes from the same registers.  The reference has no such
function; in its terms it is the row-wise fusion of
cupy/_core/_fusion_kernel.pyx:99-115, which takes one kernel per reduction.
"""
import math

import numpy

from cupy_amd._core import _op_calls as _oc
from cupy_amd._core._op_calls import Ref
from cupy_amd._core.core import ndarray

# Squares of float32 elements leave the range of float32 at 2^64 and 2^-75, and the
# gradient's powers of r before that.  With RANGED, a row whose sum of squares lies
# outside what is safe for all of them is taken again, times a power of two: the
# factor is exact, so that rows of any size have the digits of those in between.
# (Sums in 64 bits would cost every row what this costs those few: two compares are
# all that other rows see of it.)  float16 rows never leave the range.
_RANGE = r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<X_T>::type A;

#ifdef RANGED
// `low`: 0 where eps is large enough for small sums to have no say in r.  (False for a
// NaN.)
_CUPY_DEV bool out_of_range(float square, float low) {
  return (square > 0x1p80f) | (square < low);
}
// The power of two that brings the larger of `top`, the row's largest magnitude, and
// `root`, the root of eps, near 1; an infinity stays one.
_CUPY_DEV float scale_for(float top, float root) {
  const unsigned int b = __builtin_bit_cast(unsigned int, __builtin_fmaxf(top, root)) >> 23;
  return cupy::from_bits((254u - (b < 1 ? 1 : b > 253 ? 253 : b)) << 23);
}
// eps for a row times f
_CUPY_DEV float scaled_eps(double eps, float f) { return static_cast<float>(eps * f * f); }
#endif
'''

_SOURCE = _oc.Source(_RANGE + r'''
typedef cupy::bits_of<A>::type Bits;

struct Stat { A square; Bits top; };
struct JoinStat {
  _CUPY_DEV Stat operator()(const Stat& a, const Stat& b) const {
    Stat r;
    r.square = a.square + b.square;
    r.top = a.top > b.top ? a.top : b.top;
    return r;
  }
};

#ifdef INT8
typedef signed char Y_T;
#else
typedef X_T Y_T;
#endif

// What a row's statistics turn its elements h * weight into (f * h * weight with the
// statistics of the row times f).
struct Finish {
  A r, inv, lift;
  A scale;
  _CUPY_DEV Finish(const Stat& s, int width, A eps) {
    r = A(1) / cupy::sqrt_(s.square / A(width) + eps);
#ifdef INT8
    // max |y| = r * max |h w|, and q = y / scale = h w * (127 / max |h w|): r
    // cancels.  Tiny rows are lifted by a power of two first, so that the
    // quotient stays finite.
    const A top = cupy::from_bits(s.top);
    const bool tiny = top < A(1e-30);
    lift = tiny ? A(1.2676506002282294e30) : A(1);     // 2^100
    inv = top > A(0) ? A(127) / (top * lift) : A(0);
    scale = top * r / A(127);
#endif
  }
  _CUPY_DEV Y_T operator()(A hw) const {
#ifdef INT8
    // (a NaN compares false both ways and becomes 0; the row's scale is NaN)
    const A q = cupy::rint_(hw * lift * inv);
    return static_cast<signed char>(q >= A(-127) ? (q <= A(127) ? static_cast<int>(q) : 127)
                                                 : (q < A(-127) ? -127 : 0));
#else
    return static_cast<Y_T>(hw * r);
#endif
  }
};

// h of one vector, from registers.  The sum is rounded to the type it is
// stored in only on its way to memory: y follows from the unrounded sum.
template <int N>
_CUPY_DEV void sums_of(const cupy::Vec<X_T, N>& x, const cupy::Vec<R_T, N>& res, A (&h)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    h[e] = static_cast<A>(x.v[e]);
#ifdef RESIDUAL
    h[e] += static_cast<A>(res.v[e]);
#endif
  }
}

// Rows walked twice, the second time out of the cache, by kLanes lanes each, from the
// workgroup's row `base` on.  Every element is written by the thread that read it, in
// the second walk only, so outputs may lie on inputs here too.  A lane adds up what
// it would add up of a row in registers, in that order.
// A row that is out of range is walked for its largest magnitude and again, times f,
// for its statistics.
template <int kLanes>
_CUPY_DEV void walk_rows(const X_T* x, const R_T* res, const W_T* w, Y_T* y, float* scale, R_T* sum,
                         long long base, const long long rows, const int width, const long long px,
                         const long long pr, const long long py, const long long ps,
                         const double eps, const float low, const float root,
                         Stat (&lds)[2][BLOCK / 64], int flip) {
  constexpr int kRows = BLOCK / kLanes;
  const int lane = threadIdx.x % kLanes;
  for (; base < rows; base += (long long)gridDim.x * kRows) {
    const long long at = base + threadIdx.x / kLanes;
    const bool valid = kRows == 1 || at < rows;
    const long long row = valid ? at : rows - 1;
    A f = A(1), row_eps = static_cast<A>(eps);
    Stat s;
    for (bool again = false;; again = true) {
      s.square = A(0);
      s.top = 0;
      for (long long c = lane * VEC; c < width; c += kLanes * VEC) {
        const int have = width - c < VEC ? static_cast<int>(width - c) : VEC;
        const cupy::Vec<X_T, VEC> xv = cupy::load_part<X_T, VEC>(x + row * px + c, have);
        cupy::Vec<R_T, VEC> rv;
#ifdef RESIDUAL
        rv = cupy::load_part<R_T, VEC>(res + row * pr + c, have);
#endif
        A h[VEC];
        sums_of<VEC>(xv, rv, h);
        cupy::Vec<W_T, VEC> wv;
#if defined(INT8) && defined(WEIGHT)
        wv = cupy::load_part<W_T, VEC>(w + c, have);
#endif
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#ifdef RANGED
          h[e] *= f;
#endif
          s.square = cupy::fma_(h[e], h[e], s.square);
#ifdef INT8
#ifdef WEIGHT
          const Bits b = cupy::abs_bits(h[e] * static_cast<A>(wv.v[e]));
#else
          const Bits b = cupy::abs_bits(h[e]);
#endif
          s.top = b > s.top ? b : s.top;
#endif
        }
      }
      s = cupy::row_allreduce<kLanes, BLOCK>(s, JoinStat(), lds[flip]);
      flip ^= 1;
#ifdef RANGED
      if (again || !out_of_range(s.square, low)) break;
      Stat t;
      t.square = A(0);
      t.top = 0;
      for (long long c = lane; c < width; c += kLanes) {
        A h = static_cast<A>(x[row * px + c]);
#ifdef RESIDUAL
        h += static_cast<A>(res[row * pr + c]);
#endif
        const Bits b = cupy::abs_bits(h);
        t.top = b > t.top ? b : t.top;
      }
      t = cupy::row_allreduce<kLanes, BLOCK>(t, JoinStat(), lds[flip]);
      flip ^= 1;
      f = scale_for(cupy::from_bits(t.top), root);
      row_eps = scaled_eps(eps, f);
#else
      break;
#endif
    }
    const Finish fin(s, width, row_eps);
    if (!valid) continue;
    for (long long c = lane * VEC; c < width; c += kLanes * VEC) {
      const int have = width - c < VEC ? static_cast<int>(width - c) : VEC;
      const cupy::Vec<X_T, VEC> xv = cupy::load_part<X_T, VEC>(x + row * px + c, have);
      cupy::Vec<R_T, VEC> rv;
#ifdef RESIDUAL
      rv = cupy::load_part<R_T, VEC>(res + row * pr + c, have);
#endif
      A h[VEC];
      sums_of<VEC>(xv, rv, h);
#ifdef RESIDUAL
      cupy::Vec<R_T, VEC> hv;
#pragma unroll
      for (int e = 0; e < VEC; ++e) hv.v[e] = static_cast<R_T>(h[e]);
      cupy::store_part<R_T, VEC>(sum + row * ps + c, hv, have);
#endif
#ifdef RANGED
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[e] *= f;
#endif
      cupy::Vec<Y_T, VEC> yv;
#ifdef WEIGHT
      const cupy::Vec<W_T, VEC> wv = cupy::load_part<W_T, VEC>(w + c, have);
#pragma unroll
      for (int e = 0; e < VEC; ++e) yv.v[e] = fin(h[e] * static_cast<A>(wv.v[e]));
#else
#pragma unroll
      for (int e = 0; e < VEC; ++e) yv.v[e] = fin(h[e]);
#endif
      cupy::store_part<Y_T, VEC>(y + row * py + c, yv, have);
    }
#ifdef INT8
    if (lane == 0) scale[row] = static_cast<float>(fin.scale);
#endif
  }
}

#if ITEMS > 0
// Bound by memory (9001 x 2047 float32 with residual: 50.5 us, 5.8 TB/s; 4096 x
// 8192 float16 to int8: 48 us, 4.9 TB/s, where two workgroups fill a unit).
#ifdef WAVES
extern "C" __global__ void __launch_bounds__(BLOCK, WAVES)
#else
extern "C" __global__ void __launch_bounds__(BLOCK)
#endif
cupy_rms_norm(const X_T* x, const R_T* res, const W_T* w, Y_T* y, float* scale, R_T* sum,
              const long long rows, const int width, const long long px, const long long pr,
              const long long py, const long long ps, const double eps, const float low,
              const float root) {
  constexpr int kRows = BLOCK / LANES;
  __shared__ Stat lds[2][BLOCK / 64];
  const cupy::RowShare<ITEMS, LANES, VEC, TINY> mine(threadIdx.x % LANES, width);
  cupy::Vec<W_T, VEC> wv[ITEMS];
#ifdef WEIGHT
  mine.load(wv, w);
#endif
  int flip = 0;
  long long base = (long long)blockIdx.x * kRows;
  for (; base < rows; base += (long long)gridDim.x * kRows) {
    const long long at = base + threadIdx.x / LANES;
    const bool valid = kRows == 1 || at < rows;
    const long long row = valid ? at : rows - 1;
    cupy::Vec<X_T, VEC> xv[ITEMS];
    cupy::Vec<R_T, VEC> rv[ITEMS];
    mine.template load<NT_IN>(xv, x + row * px);
#ifdef RESIDUAL
    mine.template load<NT_IN>(rv, res + row * pr);
#endif
    Stat s;
    s.square = A(0);
    s.top = 0;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      A h[VEC];
      sums_of<VEC>(xv[k], rv[k], h);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (!mine.owns(k, e)) h[e] = A(0);
        s.square = cupy::fma_(h[e], h[e], s.square);
#ifdef INT8
#ifdef WEIGHT
        // (what is not owned counts as 0 whatever the weight is)
        const Bits b = cupy::abs_bits(mine.owns(k, e) ? h[e] * static_cast<A>(wv[k].v[e]) : A(0));
#else
        const Bits b = cupy::abs_bits(h[e]);
#endif
        s.top = b > s.top ? b : s.top;
#endif
      }
    }
    s = cupy::row_allreduce<LANES, BLOCK>(s, JoinStat(), lds[flip]);
    flip ^= 1;
#ifdef RANGED
    // (rows that share a wave go together, and so do all that the wave has left: a way
    // back would cost the rows in range registers)
    if (__ballot(out_of_range(s.square, low)) != 0) break;
#endif
    const Finish fin(s, width, static_cast<A>(eps));
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (!valid || !mine.any(k)) continue;
      A h[VEC];
      sums_of<VEC>(xv[k], rv[k], h);
#ifdef RESIDUAL
      cupy::Vec<R_T, VEC> hv;
#pragma unroll
      for (int e = 0; e < VEC; ++e) hv.v[e] = static_cast<R_T>(h[e]);
      mine.template store<NT_OUT>(k, sum + row * ps, hv);
#endif
      cupy::Vec<Y_T, VEC> yv;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
#ifdef WEIGHT
        yv.v[e] = fin(h[e] * static_cast<A>(wv[k].v[e]));
#else
        yv.v[e] = fin(h[e]);
#endif
      }
      mine.template store<NT_Y>(k, y + row * py, yv);
    }
#ifdef INT8
    if (valid && threadIdx.x % LANES == 0) scale[row] = static_cast<float>(fin.scale);
#endif
  }
#ifdef RANGED
  walk_rows<LANES>(x, res, w, y, scale, sum, base, rows, width, px, pr, py, ps, eps, low, root, lds,
                   flip);
#endif
}
#else
// Rows longer than the registers hold.
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_rms_norm(const X_T* x, const R_T* res, const W_T* w, Y_T* y, float* scale, R_T* sum,
              const long long rows, const int width, const long long px, const long long pr,
              const long long py, const long long ps, const double eps, const float low,
              const float root) {
  __shared__ Stat lds[2][BLOCK / 64];
  walk_rows<BLOCK>(x, res, w, y, scale, sum, blockIdx.x, rows, width, px, pr, py, ps, eps, low, root,
                   lds, 0);
}
#endif
''')

_GRAD_SOURCE = _oc.Source(_RANGE + r'''
struct Pair { A square, dot; };
struct JoinPair {
  _CUPY_DEV Pair operator()(const Pair& a, const Pair& b) const {
    Pair r;
    r.square = a.square + b.square;
    r.dot = a.dot + b.dot;
    return r;
  }
};

// With n = x r, a = g w and m = mean(a n):  dx = r (a - n m) = r a - x k,
// k = r^3 sum(a x) / width;  dw = sum over the rows of g n.  The sum is as large as
// r is small: r is multiplied to it one by one, for r^3 alone leaves the range of
// float32 from rows of 1e13 (and 1e-13) on, where k does not.  With the sums of a row
// times f: dx = f (r a - f x k), n = f x r.
struct Factors {
  A r, k;
  _CUPY_DEV Factors(const Pair& s, int width, A eps) {
    r = A(1) / cupy::sqrt_(s.square / A(width) + eps);
    k = r * (r * (r * (s.dot / A(width))));
  }
};

// What a row's n is made of, in one word: x times r (with the sums of x), or, where
// f r may be no number of the type, -(f r) 2^-64 or -(f r) 2^64, whichever f is far from.
_CUPY_DEV A factor_of(A r, A f) {
#ifdef RANGED
  if (f > 0x1p100f) return -(f * 0x1p-64f * r);
  if (f < 0x1p-100f) return -(f * 0x1p64f * r);
#endif
  return f * r;
}
_CUPY_DEV A normalised(X_T x, A factor) {
#ifdef RANGED
  const A by = factor < A(0) ? (factor > A(-1) ? A(0x1p-64f) : A(0x1p64f)) : A(1);
  return static_cast<A>(x) * by * cupy::abs_(factor);
#else
  return static_cast<A>(x) * factor;
#endif
}

#ifdef RANGED
struct LargerSquare {
  _CUPY_DEV Pair operator()(const Pair& a, const Pair& b) const {
    return a.square > b.square ? a : b;
  }
};
// (also where only the products with a are too large)
_CUPY_DEV bool out_of_range(const Pair& s, float low) {
  return out_of_range(s.square, low) | !(cupy::abs_(s.dot) < __builtin_inff());
}
#endif

// Rows walked twice by the whole workgroup, from its row `base` on: a thread adds up
// what it would of a row in registers, in that order, and writes what it read.  A row
// that is out of range is walked for its largest magnitude and again, times f.
// `factors` (if any) receives what the rows' n are made of, `dw` (if any) is added to.
_CUPY_DEV void walk_rows(const X_T* g, const X_T* x, const W_T* w, const R_T* dres, X_T* dx,
                         A* factors, A* dw, long long base, const long long rows, const int width,
                         const long long pg, const long long px, const long long pr,
                         const long long pd, const double eps, const float low, const float root,
                         Pair (&lds)[2][BLOCK / 64], int flip) {
  for (long long row = base; row < rows; row += gridDim.x) {
    A f = A(1), row_eps = static_cast<A>(eps);
    Pair s;
    for (bool again = false;; again = true) {
      s.square = s.dot = A(0);
      for (long long c = (long long)threadIdx.x * VEC; c < width; c += BLOCK * VEC) {
        const int have = width - c < VEC ? static_cast<int>(width - c) : VEC;
        const cupy::Vec<X_T, VEC> xv = cupy::load_part<X_T, VEC>(x + row * px + c, have);
        const cupy::Vec<X_T, VEC> gv = cupy::load_part<X_T, VEC>(g + row * pg + c, have);
        cupy::Vec<W_T, VEC> wv;
#ifdef WEIGHT
        wv = cupy::load_part<W_T, VEC>(w + c, have);
#endif
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#ifdef RANGED
          const A xe = static_cast<A>(xv.v[e]) * f;
#else
          const A xe = static_cast<A>(xv.v[e]);
#endif
          A a = static_cast<A>(gv.v[e]);
#ifdef WEIGHT
          a *= static_cast<A>(wv.v[e]);
#endif
          s.square = cupy::fma_(xe, xe, s.square);
          s.dot = cupy::fma_(a, xe, s.dot);
        }
      }
      s = cupy::row_allreduce<BLOCK, BLOCK>(s, JoinPair(), lds[flip]);
      flip ^= 1;
#ifdef RANGED
      if (again || !out_of_range(s, low)) break;
      Pair t;
      t.square = t.dot = A(0);
      for (long long c = threadIdx.x; c < width; c += BLOCK) {
        const A m = cupy::abs_(static_cast<A>(x[row * px + c]));
        t.square = m > t.square ? m : t.square;
      }
      t = cupy::row_allreduce<BLOCK, BLOCK>(t, LargerSquare(), lds[flip]);
      flip ^= 1;
      f = scale_for(t.square, root);
      row_eps = scaled_eps(eps, f);
#else
      break;
#endif
    }
    const Factors fac(s, width, row_eps);
    if (factors && threadIdx.x == 0) factors[row] = factor_of(fac.r, f);
    for (long long c = (long long)threadIdx.x * VEC; c < width; c += BLOCK * VEC) {
      const int have = width - c < VEC ? static_cast<int>(width - c) : VEC;
      const cupy::Vec<X_T, VEC> xv = cupy::load_part<X_T, VEC>(x + row * px + c, have);
      const cupy::Vec<X_T, VEC> gv = cupy::load_part<X_T, VEC>(g + row * pg + c, have);
      cupy::Vec<W_T, VEC> wv;
#ifdef WEIGHT
      wv = cupy::load_part<W_T, VEC>(w + c, have);
#endif
      cupy::Vec<R_T, VEC> rv;
#ifdef RESIDUAL
      rv = cupy::load_part<R_T, VEC>(dres + row * pr + c, have);
#endif
      cupy::Vec<X_T, VEC> d;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        A xe = static_cast<A>(xv.v[e]);
        const A ge = static_cast<A>(gv.v[e]);
        A a = ge;
#ifdef WEIGHT
        a *= static_cast<A>(wv.v[e]);
#endif
#ifdef RANGED
        xe *= f;
        if (dw && e < have) dw[c + e] = cupy::fma_(ge, xe * fac.r, dw[c + e]);
#endif
        A v = cupy::fma_(-xe, fac.k, a * fac.r);
#ifdef RANGED
        v *= f;
#endif
#ifdef RESIDUAL
        v += static_cast<A>(rv.v[e]);
#endif
        d.v[e] = static_cast<X_T>(v);
      }
      cupy::store_part<X_T, VEC>(dx + row * pd + c, d, have);
    }
  }
}

#if ITEMS > 0
// Bound by memory (16384 x 4096 float16 with residual: 97 us, 5.5 TB/s).
// FEW: what every row's n is made of is kept, for dw by a kernel of its own.
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_rms_norm_grad(const X_T* g, const X_T* x, const W_T* w, const R_T* dres, X_T* dx,
                   A* partial, const long long rows, const int width, const long long pg,
                   const long long px, const long long pr, const long long pd, const double eps,
                   const float low, const float root) {
  constexpr int kRows = BLOCK / LANES;
  __shared__ Pair lds[2][BLOCK / 64];
  const int lane = threadIdx.x % LANES;
  const cupy::RowShare<ITEMS, LANES, VEC, TINY> mine(lane, width);
#ifdef WEIGHT
  cupy::Vec<W_T, VEC> wv[ITEMS];
  mine.load(wv, w);
#ifndef FEW
  A dw[ITEMS][VEC];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[k][e] = A(0);
#endif
#endif
  int flip = 0;
  long long base = (long long)blockIdx.x * kRows;
  for (; base < rows; base += (long long)gridDim.x * kRows) {
    const long long at = base + threadIdx.x / LANES;
    const bool valid = kRows == 1 || at < rows;
    const long long row = valid ? at : rows - 1;
    cupy::Vec<X_T, VEC> xv[ITEMS], gv[ITEMS];
    cupy::Vec<R_T, VEC> rv[ITEMS];
    mine.template load<NT_IN>(xv, x + row * px);
    mine.template load<NT_IN>(gv, g + row * pg);
#ifdef RESIDUAL
    mine.template load<NT_IN>(rv, dres + row * pr);
#endif
    Pair s;
    s.square = s.dot = A(0);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const A xe = mine.owns(k, e) ? static_cast<A>(xv[k].v[e]) : A(0);
        A a = mine.owns(k, e) ? static_cast<A>(gv[k].v[e]) : A(0);
#ifdef WEIGHT
        a = mine.owns(k, e) ? a * static_cast<A>(wv[k].v[e]) : A(0);
#endif
        s.square = cupy::fma_(xe, xe, s.square);
        s.dot = cupy::fma_(a, xe, s.dot);
      }
    }
    s = cupy::row_allreduce<LANES, BLOCK>(s, JoinPair(), lds[flip]);
    flip ^= 1;
    A scale = A(1), row_eps = static_cast<A>(eps);
#ifdef RANGED
    if (LANES > 64) {
      // (all that the workgroup has left is walked: a way back would cost the rows in
      // range registers)
      if (__ballot(out_of_range(s, low)) != 0) break;
    } else if (__builtin_expect(out_of_range(s, low), 0)) {
      // (a lane holds one vector of the row)
      Pair t;
      t.square = t.dot = A(0);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const A m = mine.owns(0, e) ? cupy::abs_(static_cast<A>(xv[0].v[e])) : A(0);
        t.square = m > t.square ? m : t.square;
      }
      t = cupy::row_allreduce<LANES, BLOCK>(t, LargerSquare(), lds[flip]);
      scale = scale_for(t.square, root);
      row_eps = scaled_eps(eps, scale);
      s.square = s.dot = A(0);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const A xe = mine.owns(0, e) ? static_cast<A>(xv[0].v[e]) * scale : A(0);
        A a = mine.owns(0, e) ? static_cast<A>(gv[0].v[e]) : A(0);
#ifdef WEIGHT
        a = mine.owns(0, e) ? a * static_cast<A>(wv[0].v[e]) : A(0);
#endif
        s.square = cupy::fma_(xe, xe, s.square);
        s.dot = cupy::fma_(a, xe, s.dot);
      }
      s = cupy::row_allreduce<LANES, BLOCK>(s, JoinPair(), lds[flip]);
    }
#endif
    if (!valid) continue;
    const Factors f(s, width, row_eps);
#ifdef FEW
    if (threadIdx.x == 0) partial[row] = f.r;
#endif
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (!mine.any(k)) continue;
      cupy::Vec<X_T, VEC> d;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        A xe = static_cast<A>(xv[k].v[e]);
        const A ge = static_cast<A>(gv[k].v[e]);
#ifdef RANGED
        if (LANES <= 64) xe *= scale;
#endif
        A a = ge;
#ifdef WEIGHT
        a *= static_cast<A>(wv[k].v[e]);
#ifndef FEW
        dw[k][e] = cupy::fma_(ge, xe * f.r, dw[k][e]);
#endif
#endif
        A v = cupy::fma_(-xe, f.k, a * f.r);
#ifdef RANGED
        if (LANES <= 64) v *= scale;
#endif
#ifdef RESIDUAL
        v += static_cast<A>(rv[k].v[e]);
#endif
        d.v[e] = static_cast<X_T>(v);
      }
      mine.template store<NT_OUT>(k, dx + row * pd, d);
    }
  }
#if defined(WEIGHT) && !defined(FEW)
  // the workgroup's share of dw: its groups of lanes are added in order
  if (kRows == 1) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (mine.owns(k, e)) partial[(long long)blockIdx.x * width + mine.at[k] + e] = dw[k][e];
    }
  } else {
    __shared__ A shares[kRows == 1 ? 1 : BLOCK * VEC];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      __syncthreads();
      // (the elements in their own places, not in those they were loaded from)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (mine.owns(k, e)) shares[threadIdx.x * VEC + e - mine.skip[k]] = dw[k][e];
      __syncthreads();
      for (int i = threadIdx.x; i < LANES * VEC; i += BLOCK) {
        const int c = k * LANES * VEC + i;
        if (c >= width) break;
        A t = A(0);
        for (int q = 0; q < kRows; ++q) t += shares[q * LANES * VEC + i];
        partial[(long long)blockIdx.x * width + c] = t;
      }
    }
  }
#endif
#ifdef RANGED
  if (LANES > 64) {
#if defined(FEW)
    A *factors = partial, *sums = nullptr;
#elif defined(WEIGHT)
    // (every column's sum is one thread's, here and above)
    A *factors = nullptr, *sums = partial + (long long)blockIdx.x * width;
#else
    A *factors = nullptr, *sums = nullptr;
#endif
    walk_rows(g, x, w, dres, dx, factors, sums, base, rows, width, pg, px, pr, pd, eps, low, root,
              lds, flip);
  }
#endif
}
#else
// Rows longer than the registers hold; what their n are made of is kept for the sums
// down the columns, which a kernel of their own makes.
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_rms_norm_grad(const X_T* g, const X_T* x, const W_T* w, const R_T* dres, X_T* dx,
                   A* factors, const long long rows, const int width, const long long pg,
                   const long long px, const long long pr, const long long pd, const double eps,
                   const float low, const float root) {
  __shared__ Pair lds[2][BLOCK / 64];
  walk_rows(g, x, w, dres, dx, factors, nullptr, blockIdx.x, rows, width, pg, px, pr, pd, eps, low,
            root, lds, 0);
}
#endif

// Partial sum of dw over the p-th run of rows, a thread per column: the first
// `skip` words of `temp` are what the rows' n are made of, the partial sums follow.
extern "C" __global__ void __launch_bounds__(256)
cupy_rms_norm_columns(const X_T* g, const X_T* x, A* temp, const long long rows,
                      const int width, const long long pg, const long long px,
                      const long long run, const long long skip) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  const long long r0 = blockIdx.y * run;
  const long long r1 = r0 + run < rows ? r0 + run : rows;
  A t = A(0);
  for (long long r = r0; r < r1; ++r)
    t = cupy::fma_(static_cast<A>(g[r * pg + c]), normalised(x[r * px + c], temp[r]), t);
  temp[skip + (long long)blockIdx.y * width + c] = t;
}

// dw of few rows from what the rows were made of, which the caches still hold, and
// their factors: 64 columns by 16 slices of the rows to a workgroup, each slice in order,
// the slices by a tree (300 x 12000 float16: 14.7 us in all; 27 with partial rows).
extern "C" __global__ void __launch_bounds__(1024)
cupy_rms_norm_few(const X_T* g, const X_T* x, const A* factors, W_T* dw, const int rows,
                  const int width, const long long pg, const long long px) {
  constexpr int kAhead = 8, kSlices = 16;
  __shared__ A lds[kSlices][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, from = c < width ? c : width - 1;
  A t = A(0);
  for (int r0 = slice; r0 < rows; r0 += kSlices * kAhead) {
    X_T gv[kAhead], xv[kAhead];
    A rv[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = r0 + kSlices * k < rows ? r0 + kSlices * k : rows - 1;
      gv[k] = g[r * pg + from];
      xv[k] = x[r * px + from];
      rv[k] = factors[r];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (r0 + kSlices * k < rows)
        t = cupy::fma_(static_cast<A>(gv[k]), normalised(xv[k], rv[k]), t);
  }
  lds[slice][lane] = t;
  __syncthreads();
#pragma unroll
  for (int half = kSlices / 2; half > 0; half >>= 1) {
    if (slice < half) lds[slice][lane] += lds[slice + half][lane];
    __syncthreads();
  }
  if (slice == 0 && c < width) dw[c] = static_cast<W_T>(lds[0][lane]);
}

// dw = the sum of the partial rows: 32 columns (a cache line of float32) by 32
// slices of the partial rows to a workgroup; a slice is summed in order, the
// slices by a tree.  768 rows of 4096: 4.7 us, three waits in a chain.
extern "C" __global__ void __launch_bounds__(1024)
cupy_rms_norm_join(const A* temp, W_T* dw, const long long skip, const int n, const int width) {
  constexpr int kAhead = 8;
  __shared__ A lds[32][33];
  const A* partial = temp + skip;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  A t = A(0);
  if (c < width) {
    for (int p = ty; p < n; p += 32 * kAhead) {
      A v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        v[k] = partial[(long long)(p + 32 * k < n ? p + 32 * k : p) * width + c];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) if (p + 32 * k < n) t += v[k];
    }
  }
  lds[ty][tx] = t;
  __syncthreads();
#pragma unroll
  for (int half = 16; half > 0; half >>= 1) {
    if (ty < half) lds[ty][tx] += lds[ty + half][tx];
    __syncthreads();
  }
  if (ty == 0 && c < width) dw[c] = static_cast<W_T>(lds[0][tx]);
}
''')

_plans = {}
_plans_int8 = {}
_plans_grad = {}

def _geometry(width, itemsize, most_items):
    """(lanes per row, threads of a workgroup, vectors per lane, elements per
    vector) of rows held in registers; 0 vectors: too long for them.

    One vector per lane, as many lanes as that takes: all of a row is requested
    at once and the units hold many rows (16384 x 4096 float16 with residual:
    89 us with 512 lanes, 92 with 256 and two vectors; 9001 x 2047 float32: 50.5
    with 512, 52.8 with 256; 4096 x 8192 to int8: 66 with 1024, 75 with 512, 84
    with 256).  Rows of up to 64 vectors share a workgroup of 256 threads, longer
    ones take whole waves."""
    vec = 16 // itemsize
    n = (width + vec - 1) // vec
    if n <= 64:
        return max(4, _oc.clp2(n)), 256, 1, vec
    # as many lanes for every vector of a lane, whole waves of them
    each = -(-n // 1024)
    lanes = min(1024, -(-n // (64 * each)) * 64)
    items = -(-n // lanes)
    if items > most_items:
        return 1024, 1024, 0, vec
    return lanes, lanes, items, vec


def _range_of(eps):
    """(smallest sum of squares that is safe, root of eps) for the kernels of float32 rows."""
    return 2.0 ** -60 if eps < 2.0 ** -40 else 0.0, min(math.sqrt(eps), 1e38) if eps > 0 else 0.0


def _held_eps(dtype, ranged, eps):
    """eps for kernels that hold it in 32 bits: above 0 there too.  (The mean square of
    float16 rows is 0 or far above 1e-38; RANGED kernels take it as it is.)"""
    return 1e-38 if dtype.char != 'd' and not ranged and 0 < eps < 1e-38 else eps


def _check(x, weight, residual, what):
    _oc.check_float(x, 'x')
    if x.ndim == 0:
        raise ValueError('%s takes arrays of at least one dimension' % what)
    if x._shape[-1] >= 1 << 31:
        raise ValueError('%s: rows of 2**31 elements and more are not supported' % what)
    if weight is not None:
        _oc.check_float(weight, 'weight')
        if weight._shape != x._shape[-1:]:
            raise ValueError('weight has the wrong shape: %r, expected %r'
                             % (weight._shape, x._shape[-1:]))
        _check_mix(weight.dtype, x.dtype, 'weight')
    if residual is not None:
        _oc.check_float(residual, 'residual')
        if residual._shape != x._shape:
            raise ValueError('residual has the wrong shape: %r, expected %r'
                             % (residual._shape, x._shape))
        _check_mix(residual.dtype, x.dtype, 'residual')


def _check_mix(dtype, base, name):
    if dtype != base and not (base.char == 'e' and dtype.char == 'f'):
        raise TypeError('%s of type %s does not go with x of type %s: the type of x, or float32 '
                        'with float16' % (name, dtype, base))


def _norm(plans, int8, x, weight, residual, eps, out, scale_out, residual_out):
    eps = float(eps)
    arrays = [x]
    flags = 0
    if weight is not None:
        arrays.append(weight)
        flags = 1
    if residual is not None:
        arrays.append(residual)
        flags |= 2
    if out is not None:
        arrays.append(out)
        flags |= 4
    if scale_out is not None:
        arrays.append(scale_out)
        flags |= 8
    if residual_out is not None:
        arrays.append(residual_out)
        flags |= 16
    result, key = _oc.replay(plans, arrays, (flags, eps))
    if result is not _oc._NOTHING:
        return result
    _check(x, weight, residual, 'rms_norm')
    if residual_out is not None and residual is None:
        raise ValueError('residual_out without residual')
    y_dtype = numpy.dtype(numpy.int8) if int8 else x.dtype
    if out is not None:
        _oc.check_out(out, x._shape, y_dtype)
    if scale_out is not None:
        _oc.check_out(scale_out, x._shape[:-1], numpy.dtype(numpy.float32), 'scale_out')
    if residual_out is not None:
        _oc.check_out(residual_out, x._shape, residual.dtype, 'residual_out')
    n_in = 1 + (weight is not None) + (residual is not None)
    i_w = 1 if weight is not None else None
    i_r = n_in - 1 if residual is not None else None
    at = n_in
    i_y = i_s = i_h = None
    if out is not None:
        i_y, at = at, at + 1
    if scale_out is not None:
        i_s, at = at, at + 1
    if residual_out is not None:
        i_h, at = at, at + 1
    # a row is read whole before any of it is written, and a thread writes what
    # it read: the outputs may take the place of x and the residual
    places = [(i, o) for i in (0, i_r) if i is not None for o in (i_y, i_h) if o is not None]
    call = _oc.Call(plans, key, arrays, n_in, places)
    if i_y is None:
        i_y = call.allocate(x._shape, y_dtype)
    if int8 and i_s is None:
        i_s = call.allocate(x._shape[:-1], numpy.float32)
    if residual is not None and i_h is None:
        i_h = call.allocate(x._shape, residual.dtype)
    ret = (i_y,) + ((i_s,) if int8 else ()) + ((i_h,) if residual is not None else ())
    width = x._shape[-1]
    if x.size == 0:
        call.key = None
        if int8:
            call.refs[i_s].fill(0)
        call.begin()
        out = call.finish(ret)
        return out if len(out) > 1 else out[0]
    rows = x.size // width
    px = call.rows(0)
    pr = call.rows(i_r) if i_r is not None else 0
    py = call.rows(i_y)
    ps = call.rows(i_h) if i_h is not None else 0
    if i_w is not None:
        call.dense(i_w)
    if int8:
        call.dense(i_s)
    call.begin()
    lanes, block, items, vec = _geometry(width, x.dtype.itemsize, 4)
    nt_in, nt_out = _oc.stream_hints(
        x.nbytes + (residual.nbytes if residual is not None else 0),
        x.size * y_dtype.itemsize + (residual.nbytes if residual is not None else 0))
    defines = dict(X_T=x.dtype, R_T=x.dtype if residual is None else residual.dtype,
                   W_T=x.dtype if weight is None else weight.dtype, LANES=lanes, BLOCK=block,
                   ITEMS=items, VEC=vec, TINY=width < vec, NT_IN=nt_in, NT_OUT=nt_out,
                   # (8 bits fit the cache where the rest does not)
                   NT_Y=nt_out and not int8)
    ranged = 'f' in (x.dtype.char, defines['R_T'].char)
    for name, on in (('INT8', int8), ('WEIGHT', weight is not None),
                     ('RESIDUAL', residual is not None), ('RANGED', ranged)):
        if on:
            defines[name] = 1
    # The walks may not cost the rows in registers the second workgroup on a unit: the
    # compiler is asked for two where a lane holds few enough words of x, the weight and
    # the residual (16384 x 4096 float32 to int8: 134 us, 156 unasked; 300 x 12000: 10.6
    # and 11.1; but 400 x 16384 with residual, 48 words: 19.5 and 18.5, for some spill).
    held = items * vec * (x.dtype.itemsize
                          + (weight.dtype.itemsize if weight is not None else 0)
                          + (residual.dtype.itemsize if residual is not None else 0)) // 4
    if ranged and block > 512 and 0 < held <= 40:
        defines['WAVES'] = -(-2 * block // 256)
    fn = _SOURCE.function('cupy_rms_norm', **defines)
    # A workgroup per row (or 256 / lanes of them): stores run fastest without a
    # loop around them.  Of those of more than 512 threads a unit holds two: they
    # loop (4096 x 8192 to int8 66 us, 70 without), unless the last round of the
    # loop would leave a twentieth of them without a row.
    grid = -(-rows // (block // lanes))
    resident = 2 * _oc.compute_units()
    rounds = -(-grid // resident)
    if block > 512 and grid >= 0.95 * rounds * resident:
        grid = min(grid, resident)
    grid = min(grid, 0xffffffff // block)
    call.launch(fn, (grid, 1, 1), block, 'PPPPPPqiqqqqdff',
                Ref(0), Ref(i_r) if i_r is not None else 0, Ref(i_w) if i_w is not None else 0,
                Ref(i_y), Ref(i_s) if int8 else 0, Ref(i_h) if i_h is not None else 0,
                rows, width, px, pr, py, ps, _held_eps(x.dtype, ranged, eps), *_range_of(eps))
    out = call.finish(ret if len(ret) > 1 else ret[0])
    return out


def rms_norm(x, weight=None, residual=None, eps=1e-6, *, out=None, residual_out=None):
    """Root-mean-square norm along the last axis.

    ``y = h / sqrt(mean(h * h) + eps) * weight`` with ``h = x + residual``
    (``h = x`` without a residual).  Sums are held in 32 bits for float16 and
    float32 (64 for float64); ``y`` is rounded once, from the unrounded ``h``.
    Finite rows of float16 and float32 may be of any size; the squares of float64
    rows have to stay in its range.

    Args:
        x (cupy.ndarray): float16, float32 or float64, of one dimension or more.
        weight (cupy.ndarray): one factor per column; of the type of ``x``, or
            float32 with float16.
        residual (cupy.ndarray): added to ``x`` first; shaped like ``x``, of its
            type, or float32 with float16.
        eps (float): added to the mean square.
        out (cupy.ndarray): receives ``y``.
        residual_out (cupy.ndarray): receives ``h``, in the residual's type.

    ``out`` and ``residual_out`` may be ``x`` or ``residual`` themselves.

    Returns:
        ``y``, or ``(y, h)`` with a residual.
    """
    return _norm(_plans, False, x, weight, residual, eps, out, None, residual_out)


def rms_norm_int8(x, weight=None, residual=None, eps=1e-6, *, out=None, scale_out=None,
                  residual_out=None):
    """:func:`rms_norm` with its result in 8 bits and a scale per row.

    ``scale = max(|y|) / 127`` over the row (float32) and
    ``q = rint(y / scale)``, ties to even: ``q * scale`` is ``y`` to half a
    step.  A row of zeros has the scale 0 (``eps`` above 0); in a row with a NaN
    or an infinity the scale is NaN.

    Returns:
        ``(q, scale)``, or ``(q, scale, h)`` with a residual: int8 shaped like
        ``x``, float32 of the shape without the last axis, the sum.
    """
    return _norm(_plans_int8, True, x, weight, residual, eps, out, scale_out, residual_out)


def _start_alike(a, b):
    return isinstance(a, ndarray) and isinstance(b, ndarray) and a.data.ptr == b.data.ptr


def rms_norm_grad(grad, x, weight=None, eps=1e-6, *, residual_grad=None, out=None,
                  weight_out=None):
    """Gradients of :func:`rms_norm` with respect to its input and weight.

    With ``n = x / sqrt(mean(x * x) + eps)`` and ``a = grad * weight``:
    ``dx = (a - n * mean(a * n)) / sqrt(mean(x * x) + eps) + residual_grad`` and
    ``dw = sum of grad * n`` over all rows, in an order that does not change
    from call to call (``dx`` in the place of ``grad`` or ``x`` may have another
    order than ``dx`` elsewhere).  Rows may be as large and small as in the forward
    call.

    Args:
        grad (cupy.ndarray): gradient of ``y``, of the shape and type of ``x``.
        x (cupy.ndarray): what was normalised (``h`` where there was a residual).
        weight (cupy.ndarray): as in the forward call.
        residual_grad (cupy.ndarray): gradient that reaches ``h`` past the norm;
            of the type of ``x``, or float32 with float16.
        out (cupy.ndarray): receives ``dx``; may be ``grad``, ``x`` or
            ``residual_grad``.
        weight_out (cupy.ndarray): receives ``dw``.

    Returns:
        ``dx``, or ``(dx, dw)`` with a weight.  ``dx`` is the gradient of ``x``
        and of the residual alike.
    """
    eps = float(eps)
    arrays = [grad, x]
    flags = 0
    if weight is not None:
        arrays.append(weight)
        flags = 1
    if residual_grad is not None:
        arrays.append(residual_grad)
        flags |= 2
    if out is not None:
        arrays.append(out)
        flags |= 4
    if weight_out is not None:
        arrays.append(weight_out)
        flags |= 8
    if weight is not None and (_start_alike(out, grad) or _start_alike(out, x)):
        flags |= 16
    result, key = _oc.replay(_plans_grad, arrays, (flags, eps))
    if result is not _oc._NOTHING:
        return result
    _check(x, weight, None, 'rms_norm_grad')
    _oc.check_float(grad, 'grad')
    if grad._shape != x._shape or grad.dtype != x.dtype:
        raise ValueError('grad has to have the shape and type of x: %r %s, expected %r %s'
                         % (grad._shape, grad.dtype, x._shape, x.dtype))
    if residual_grad is not None:
        _oc.check_float(residual_grad, 'residual_grad')
        if residual_grad._shape != x._shape:
            raise ValueError('residual_grad has the wrong shape: %r, expected %r'
                             % (residual_grad._shape, x._shape))
        _check_mix(residual_grad.dtype, x.dtype, 'residual_grad')
    if weight_out is not None and weight is None:
        raise ValueError('weight_out without weight')
    if out is not None:
        _oc.check_out(out, x._shape, x.dtype)
    if weight_out is not None:
        _oc.check_out(weight_out, weight._shape, weight.dtype, 'weight_out')
    n_in = 2 + (weight is not None) + (residual_grad is not None)
    i_w = 2 if weight is not None else None
    i_r = n_in - 1 if residual_grad is not None else None
    at = n_in
    i_d = i_dw = None
    if out is not None:
        i_d, at = at, at + 1
    if weight_out is not None:
        i_dw, at = at, at + 1
    width = x._shape[-1]
    rows = x.size // width if width else 0
    lanes, block, items, vec = _geometry(width, x.dtype.itemsize, 2 if x.dtype.char == 'd' else 4)
    # Workgroups that loop over rows, each with its sums for dw in registers: of
    # 1536 threads to a unit (16384 x 4096 float16: 102 us; 107 with 2048, 111 to
    # 114 with 1024), of which each adds a partial row to what is joined.
    most = _oc.compute_units() * max(1, 1536 // block)
    # Few long rows, a workgroup to each, none of which has anything to add up: dw
    # follows from the inputs, unless dx takes their place (float16, 768 x 4096: 16.5
    # us, 19.5 with partial rows; 700 x 1003 float32: 13.9 and 11.1; 256 x 16384:
    # 18.2 and 21.8; 400 x 8192: 17.7 and 16.3).
    few = (weight is not None and items and lanes == block and rows <= most and not flags & 16
           and width >= rows * (5 if x.dtype.itemsize == 2 else 32))
    # rows in registers: written by the threads that have read them.  (Where dw
    # is a second step, that reads the inputs again.)
    places = [(i, i_d) for i in (0, 1, i_r) if i is not None and i_d is not None
              and (weight is None or i == i_r or (items and not few))]
    call = _oc.Call(_plans_grad, key, arrays, n_in, places)
    if i_d is None:
        i_d = call.allocate(x._shape, x.dtype)
    if weight is not None and i_dw is None:
        i_dw = call.allocate(weight._shape, weight.dtype)
    ret = (i_d, i_dw) if weight is not None else i_d
    if x.size == 0:
        call.key = None
        if weight is not None:
            call.refs[i_dw].fill(0)
        call.begin()
        return call.finish(ret)
    pg, px = call.rows(0), call.rows(1)
    pr = call.rows(i_r) if i_r is not None else 0
    pd = call.rows(i_d)
    if i_w is not None:
        call.dense(i_w)
        call.dense(i_dw)
    call.begin()
    nt_in, nt_out = _oc.stream_hints(3 * x.nbytes, x.nbytes)
    defines = dict(X_T=x.dtype, R_T=x.dtype if residual_grad is None else residual_grad.dtype,
                   W_T=x.dtype if weight is None else weight.dtype, LANES=lanes, BLOCK=block,
                   ITEMS=items, VEC=vec, TINY=width < vec, NT_IN=nt_in, NT_OUT=nt_out)
    for name, on in (('WEIGHT', weight is not None), ('RESIDUAL', residual_grad is not None),
                     ('RANGED', x.dtype.char == 'f')):
        if on:
            defines[name] = 1
    acc = _oc.acc_dtype(x.dtype).itemsize
    if few:
        defines['FEW'] = 1
    grid = max(1, min(-(-rows // (block // lanes)), most))
    fn = _GRAD_SOURCE.function('cupy_rms_norm_grad', **defines)
    # the temporary: a word for each row (walked rows only), then the partial sums of dw
    n_partial, skip, run = grid, 0, 0
    i_t = None
    if weight is not None:
        if not items:
            # runs of rows, about as many as keep the device busy
            blocks = -(-width // 256)
            run = -(-rows // max(1, min(rows, -(-_oc.compute_units() * 8 // blocks), 65535)))
            n_partial, skip = -(-rows // run), rows
        i_t = call.temp((rows if few else skip + n_partial * width) * acc)
    call.launch(fn, (grid, 1, 1), block, 'PPPPPPqiqqqqdff',
                Ref(0), Ref(1), Ref(i_w) if i_w is not None else 0,
                Ref(i_r) if i_r is not None else 0, Ref(i_d), Ref(i_t) if i_t is not None else 0,
                rows, width, pg, px, pr, pd, _held_eps(x.dtype, x.dtype.char == 'f', eps),
                *_range_of(eps))
    if few:
        fn = _GRAD_SOURCE.function('cupy_rms_norm_few', **defines)
        call.launch(fn, (-(-width // 64), 1, 1), 1024, 'PPPPiiqq',
                    Ref(0), Ref(1), Ref(i_t), Ref(i_dw), rows, width, pg, px)
    elif weight is not None:
        if not items:
            fn = _GRAD_SOURCE.function('cupy_rms_norm_columns', **defines)
            call.launch(fn, (blocks, n_partial, 1), 256, 'PPPqiqqqq',
                        Ref(0), Ref(1), Ref(i_t), rows, width, pg, px, run, skip)
        fn = _GRAD_SOURCE.function('cupy_rms_norm_join', **defines)
        call.launch(fn, (-(-width // 32), 1, 1), 1024, 'PPqii',
                    Ref(i_t), Ref(i_dw), skip, n_partial, width)
    return call.finish(ret)
