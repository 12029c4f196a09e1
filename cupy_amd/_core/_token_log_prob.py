"""Log probabilities of given tokens, with entropy and top alternatives, and
their gradient.

For a row of logits ``x`` and a token ``t``: ``lse = log(sum(exp(x)))``,
``log_prob = x[t] - lse``, ``entropy = -sum(p * log(p))`` with
``p = exp(x - lse)``.  All of them, and the ``top`` likeliest tokens, come from
one pass over the row with a running maximum ``m``, the sum ``s`` of
``exp(x - m)`` and, for the entropy, the sum ``u`` of ``(x - m) * exp(x - m)``:
``lse = m + log(s)``, ``entropy = log(s) - u / s``.  The reference composes
them from reductions (cupyx/scipy/special/_softmax.py, _logsumexp.py).
"""
import collections
import operator

import numpy

from cupy_amd._core import _op_calls as _oc
from cupy_amd._core._op_calls import Ref

TokenLogProb = collections.namedtuple(
    'TokenLogProb', ['log_prob', 'lse', 'entropy', 'top_log_prob', 'top_token'])
TokenLogProb.__doc__ = """What :func:`token_log_prob` returns (None where not asked for)."""

MAX_TOP = 32

_COMMON = r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<X_T>::type A;
typedef unsigned int u32;

#define LOG2E 1.4426950408889634
#define LN2 0.6931471805599453

_CUPY_DEV float exp2_(float t) { return __builtin_amdgcn_exp2f(t); }
_CUPY_DEV double exp2_(double t) { return exp2(t); }
_CUPY_DEV float max_(float a, float b) { return __builtin_fmaxf(a, b); }
_CUPY_DEV double max_(double a, double b) { return __builtin_fmax(a, b); }
template <typename T> struct lowest;
template <> struct lowest<float16> { static _CUPY_DEV A value() { return A(-65504.0f); } };
template <> struct lowest<float> { static _CUPY_DEV A value() { return A(-3.4028234663852886e38f); } };
template <> struct lowest<double> { static _CUPY_DEV A value() { return A(-1.7976931348623157e308); } };

// A row is seen as vectors of 16 bytes that start on a border of kBorder bytes,
// whatever the row starts on, and as the single elements before the first and
// behind the last of them.
template <int kBorder>
struct RowVecs {
  const X_T* x;
  int width;
  int head;         // elements before the first vector
  int n;            // vectors
  int tail;         // elements behind the last
  _CUPY_DEV RowVecs(const X_T* row, int w) : x(row), width(w) {
    const int phase =
        (int)((reinterpret_cast<unsigned long long>(row) & (kBorder - 1)) / sizeof(X_T));
    head = phase ? kBorder / (int)sizeof(X_T) - phase : 0;
    if (head > w) head = w;
    n = (w - head) / VEC;
    tail = w - head - n * VEC;
  }
  _CUPY_DEV int column(int j) const { return head + j * VEC; }
  _CUPY_DEV cupy::Vec<X_T, VEC> load(int j) const {
    return cupy::load_vec<X_T, VEC, NT_IN>(x + head + (long long)j * VEC);
  }
  // (16-byte borders) Column of the single element that thread t takes, or -1:
  // threads 0 and up the head's, threads 32 and up the tail's.
  _CUPY_DEV int single(int t) const {
    if (t < head) return t;
    if (t >= 32 && t - 32 < tail) return width - tail + t - 32;
    return -1;
  }
};

// Running statistics.  The maximum starts at the type's lowest value, not at
// -inf, so that x - m is never inf - inf: masked rows need no case of their own.
// float16: 2^(x log2e - m log2e) takes one fused multiply-add per element; the
// rounded m log2e is what is added back at the end, so its rounding cancels.
// float32: m log2e may overflow, and x - m is exact where it matters.
struct Run {
  A m, s, u;
  _CUPY_DEV static bool half() { return sizeof(X_T) == 2; }
  _CUPY_DEV A base() const { return half() ? m * A(LOG2E) : m; }
  _CUPY_DEV static A power(A x, A base) {
    return half() ? cupy::fma_(x, A(LOG2E), -base) : (x - base) * A(LOG2E);
  }
  // ... the same of another maximum, kept finite (0 * -inf)
  _CUPY_DEV A below(A to) const {
    const A d = half() ? m * A(LOG2E) - to * A(LOG2E) : (m - to) * A(LOG2E);
    return max_(d, A(-30000));
  }
  _CUPY_DEV void lift(A to) {
    const A t = below(to), f = exp2_(t);
    u = f * cupy::fma_(s, t, u);
    s *= f;
    m = to;
  }
  // one more element (-inf: nothing; its argument is kept finite for 0 * -inf)
  _CUPY_DEV void add(A x, A base) {
    const A t = power(x, base), p = exp2_(t);
    s += p;
#ifdef ENTROPY
    u = cupy::fma_(max_(t, A(-30000)), p, u);
#endif
  }
  _CUPY_DEV double log2_sum() const { return log2((double)s); }
  // What the results are made of: float16: lse; else lse - m, so that log
  // probabilities hold where m swallows it (rows of the type's lowest value).
  _CUPY_DEV double tail() const {
    constexpr double back = 1.0 / (double)A(LOG2E);
    return half() ? ((double)(m * A(LOG2E)) + log2_sum()) * back : log2_sum() * LN2;
  }
  // (s == 0: every element is -inf)
  _CUPY_DEV double lse(double tail) const {
    return s == A(0) ? -__builtin_inf() : half() ? tail : (double)m + tail;
  }
  _CUPY_DEV double log_prob(A x, double tail) const {
    if (s == A(0)) return (double)x;                 // (-inf, not NaN)
    return half() ? (double)x - tail : ((double)x - (double)m) - tail;
  }
  _CUPY_DEV double entropy() const {
    if (s == A(0)) return 0.0;
    return (log2_sum() - (double)u / (double)s) * LN2;
  }
};
struct Greater { _CUPY_DEV A operator()(A a, A b) const { return max_(a, b); } };
struct Add { _CUPY_DEV A operator()(A a, A b) const { return a + b; } };
// Joined over groups of kGroup lanes: the maximum first, so that every lane
// rescales its sums once.
template <int kGroup>
_CUPY_DEV Run join_lanes(Run r) {
  r.lift(cupy::group_allreduce<kGroup>(r.m, Greater()));
  r.s = cupy::group_allreduce<kGroup>(r.s, Add());
  r.u = cupy::group_allreduce<kGroup>(r.u, Add());
  return r;
}

// The largest element of a vector, NaNs left out.
_CUPY_DEV A largest(const cupy::Vec<X_T, VEC>& v) {
  if (sizeof(X_T) == 2) {
    // two halves at a time
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    half2 p[VEC / 2];
    __builtin_memcpy(p, &v, sizeof(p));
    half2 m = p[0];
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) m = __builtin_elementwise_max(m, p[i]);
    return max_(static_cast<A>(m.x), static_cast<A>(m.y));
  }
  A m = static_cast<A>(v.v[0]);
#pragma unroll
  for (int i = 1; i < VEC; ++i) m = max_(m, static_cast<A>(v.v[i]));
  return m;
}

#if TOP > 0
// A value and its column in one order: larger values first, of equal values the
// lower column.  float16 and float32: one word, the value's bits turned so that
// they order as integers (-0 as 0) above the complement of the column.  A key
// that stands for nothing comes behind every element, also behind -inf.
#if SMALL_KEYS
typedef unsigned long long Key;
_CUPY_DEV Key key_of(A v, u32 column) {
  const u32 b = __builtin_bit_cast(u32, v + 0.0f);
  const u32 turned = b ^ ((u32)((int)b >> 31) | 0x80000000u);
  return (Key)turned << 32 | (u32)~column;
}
_CUPY_DEV Key no_key(u32 number) { return number; }
_CUPY_DEV bool is_none(Key k) { return (k >> 32) == 0; }
_CUPY_DEV bool better(Key a, Key b) { return a > b; }
_CUPY_DEV A value_of(Key k) {
  const u32 t = (u32)(k >> 32);
  return __builtin_bit_cast(A, t & 0x80000000u ? t ^ 0x80000000u : ~t);
}
_CUPY_DEV u32 column_of(Key k) { return ~(u32)k; }
#else
struct Key {
  A v;
  u32 i;
  u32 pad;
};
_CUPY_DEV Key key_of(A v, u32 column) {
  Key k;
  k.v = v;
  k.i = column;
  k.pad = 0;
  return k;
}
_CUPY_DEV Key no_key(u32 number) { return key_of(-__builtin_inf(), 0xffffffffu - number); }
_CUPY_DEV bool is_none(const Key& k) { return k.i >= 0x80000000u; }
_CUPY_DEV bool better(const Key& a, const Key& b) {
  return (a.v > b.v) | ((a.v == b.v) & (a.i < b.i));
}
_CUPY_DEV A value_of(const Key& k) { return k.v; }
_CUPY_DEV u32 column_of(const Key& k) { return k.i; }
#endif

struct BestKey {
  _CUPY_DEV Key operator()(const Key& a, const Key& b) const {
    return cupy::select_value(better(b, a), b, a);
  }
};

_CUPY_DEV Key key_at(const cupy::Vec<X_T, VEC>& v, int j, int i, const RowVecs<16>& vecs) {
  return key_of(static_cast<A>(v.v[i]), (u32)(vecs.column(j) + i));
}

// kMost: keys that are ranked against each other
template <int kMost_>
struct TopState {
  static constexpr int kMost = kMost_;
  Key sample[64];               // (no two alike)
  Key key[kMost];
  Key last;
  double tail;
  u32 n;
};

// The TOP-th best of the 64 sample keys: at least TOP keys are as good.
template <typename State>
_CUPY_DEV Key bar(const State& t) {
  const Key me = t.sample[threadIdx.x & 63];
  int rank = 0;
#pragma unroll 8
  for (int o = 0; o < 64; ++o) rank += better(t.sample[o], me);
  return cupy::shfl_idx(me, __ffsll(__ballot(rank == TOP - 1)) - 1);
}

// The value that an element as good as `least` has at least.
_CUPY_DEV A value_at_least(const Key& least) {
  return is_none(least) ? -__builtin_inff() : value_of(least);
}
// Keeps an element that is as good as `least`, whose value is `enough` (a NaN is
// none: its row has no order).  The values are compared first: few pass.
template <typename State>
_CUPY_DEV void offer(State& t, A value, u32 column, const Key& least, A enough) {
  if (!(value >= enough)) return;
  const Key k = key_of(value, column);
  if (better(least, k)) return;
  const u32 at = atomicAdd(&t.n, 1u);
  if (at < State::kMost) t.key[at] = k;
}
#endif
'''

_SOURCE = _oc.Source(_COMMON + r'''
#if TOP > 0
// Writes the n <= kMost keys collected in t by rank, the best TOP of them.
template <typename State, typename Put>
_CUPY_DEV void put_ranked(const State& t, u32 n, Put put) {
  for (u32 q = threadIdx.x; q < n; q += blockDim.x) {
    const Key me = t.key[q];
    int rank = 0;
#pragma unroll 4
    for (u32 o = 0; o < n; ++o) rank += better(t.key[o], me);
    if (rank < TOP) put(rank, me);
  }
  // (fewer elements than TOP: the rest of the places hold nothing)
  for (u32 q = n + threadIdx.x; q < TOP; q += blockDim.x) put(q, no_key(0));
}
#endif

struct Outputs {
  A* log_prob;
  A* lse;
  A* entropy;
  A* top;
  long long* index;
};

// The logit of the row's token, 0 if it has none.
_CUPY_DEV A logit_of(const X_T* x, long long token, int width) {
  return token >= 0 && token < width ? static_cast<A>(x[token]) : A(0);
}

// A row's results from its joined statistics, by one thread.
_CUPY_DEV void put_row(const Outputs& o, const Run& run, double tail, A logit, long long token,
                       long long row, int width) {
  o.lse[row] = static_cast<A>(run.lse(tail));
  double lp = 0.0;
  if (token >= 0 && token < width) lp = run.log_prob(logit, tail);
  o.log_prob[row] = static_cast<A>(lp);
#ifdef ENTROPY
  o.entropy[row] = static_cast<A>(run.entropy());
#endif
}
#if TOP > 0
_CUPY_DEV void put_top(const Outputs& o, const Run& run, double tail, long long row, int rank,
                       const Key& k) {
  const bool nan = !(run.s == run.s);          // no order in a row with NaN or +inf
  o.top[row * TOP + rank] =
      nan ? static_cast<A>(run.s) : static_cast<A>(run.log_prob(value_of(k), tail));
  o.index[row * TOP + rank] = nan ? -1 : (long long)column_of(k);
}
#endif

// A workgroup per part of a row (PARTS == 1: the whole row, with its results).
// Bound by memory: a vector costs a compare of its maximum, and per element a
// multiply-add, an exponential (a quarter of the rate) and one or two
// additions; the rescaling by a new maximum is taken only when a vector has one.
// 8192 x 50257 float16 with entropy: 130 us, 6.3 TB/s.
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_token_log_prob(const X_T* logits, const I_T* tokens, A* log_prob, A* lse, A* entropy, A* top,
                    long long* index, A* runs, const long long rows, const int width,
                    const long long pitch, const int parts, const long long at_keys) {
  constexpr int kWaves = BLOCK / 64;
  __shared__ Run lds[kWaves];
#if TOP > 0
  constexpr int kMost = TOP == 1 ? 1 : BLOCK < 256 ? 4 * BLOCK : 1024;
  __shared__ TopState<kMost> ts;
#endif
  Outputs out;
  out.log_prob = log_prob;
  out.lse = lse;
  out.entropy = entropy;
  out.top = top;
  out.index = index;
  for (long long w = blockIdx.x; w < rows * parts; w += gridDim.x) {
    const long long row = parts == 1 ? w : w / parts;
    const int part = parts == 1 ? 0 : (int)(w - row * parts);
    const X_T* x = logits + row * pitch;
    const RowVecs<16> vecs(x, width);
    const int share = (vecs.n + parts - 1) / parts;
    const int j0 = part * share;
    const int j1 = j0 + share < vecs.n ? j0 + share : vecs.n;
    const int single = part == 0 ? vecs.single(threadIdx.x) : -1;
    Run run;
    run.m = lowest<X_T>::value();
    run.s = run.u = A(0);
    const X_T alone = x[single >= 0 ? single : 0];
    const long long token = parts == 1 ? (long long)tokens[row] : 0;
#if TOP > 0
    A best = -__builtin_inff();
    int best_at = j0 + threadIdx.x;
    const bool once = j1 - j0 <= BLOCK * UNROLL;   // one trip: its vectors stay in registers
#endif
    A base = run.base();
    cupy::Vec<X_T, VEC> v[UNROLL];
    // All vectors of a trip are requested before the first is used; the last
    // trip's requests beyond the end go to the last vector and are not used.
    for (int j = j0; j < j1; j += BLOCK * UNROLL) {
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        const int at = j + k * BLOCK + (int)threadIdx.x;
        v[k] = vecs.load(at < j1 ? at : j1 - 1);
      }
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        if (j + k * BLOCK + (int)threadIdx.x >= j1) break;
        const A vm = largest(v[k]);
#if TOP > 0
        if (vm > best) {
          best = vm;
          best_at = j + k * BLOCK + threadIdx.x;
        }
#endif
        if (vm > run.m) {
          run.lift(vm);
          base = run.base();
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) run.add(static_cast<A>(v[k].v[i]), base);
      }
    }
    if (single >= 0) {
      const A e = static_cast<A>(alone);
      if (e > run.m) run.lift(e);
      run.add(e, run.base());
    }
    const A logit = parts == 1 && threadIdx.x == 0 ? logit_of(x, token, width) : A(0);
    run = join_lanes<64>(run);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = run;
#if TOP > 0
    // The best of every thread, then of 64 groups of threads.
    Key mine = no_key(0), most = no_key(0);
    if (best_at < j1) {
#if TOP == 1
      cupy::Vec<X_T, VEC> from = v[0];
      if (once) {
#pragma unroll
        for (int k = 1; k < UNROLL; ++k)
          from = cupy::select_value(best_at == j0 + k * BLOCK + (int)threadIdx.x, v[k], from);
      } else {
        from = vecs.load(best_at);
      }
      int at = -1;
#pragma unroll
      for (int i = VEC - 1; i >= 0; --i)
        if (static_cast<A>(from.v[i]) == best) at = i;
      if (at >= 0) mine = key_of(best, (u32)(vecs.column(best_at) + at));
#else
      // Which element of its vector it is stays open, so that nothing is loaded:
      // the key is `mine` at least and `most` at most.
      mine = key_of(best, (u32)(vecs.column(best_at) + VEC - 1));
      most = key_of(best, (u32)vecs.column(best_at));
#endif
    }
    Key other = no_key(0);
    if (single >= 0 && alone == alone) {
      other = key_of(static_cast<A>(alone), (u32)single);
      mine = BestKey()(mine, other);
      most = BestKey()(most, other);
    }
    const Key group = cupy::group_allreduce<kWaves>(mine, BestKey());
    if (threadIdx.x % kWaves == 0)
      ts.sample[threadIdx.x / kWaves] = is_none(group) ? no_key(threadIdx.x / kWaves) : group;
    if (threadIdx.x == 0) ts.n = 0;
#endif
    __syncthreads();
    run = join_lanes<kWaves>(lds[threadIdx.x & (kWaves - 1)]);
    if (threadIdx.x == 0) {
      if (parts == 1) {
        const double tail = run.tail();
        put_row(out, run, tail, logit, token, row, width);
#if TOP > 0
        ts.tail = tail;
#endif
      } else {
        A* to = runs + w * 3;
        to[0] = run.m;
        to[1] = run.s;
        to[2] = run.u;
      }
    }
#if TOP > 0
    Key* keys = reinterpret_cast<Key*>(runs + at_keys) + w * TOP;
    auto put = [&](int rank, const Key& k) {
      if (parts == 1) {
        put_top(out, run, ts.tail, row, rank, k);
      } else {
        keys[rank] = k;
      }
    };
#if TOP == 1
    if (threadIdx.x < 64) {
      const Key b = cupy::group_allreduce<64>(ts.sample[threadIdx.x], BestKey());
      if (threadIdx.x == 0) put(0, b);
    }
#else
    // (one wave finds the bar: what every wave does here costs the most of it)
    if (kWaves > 1) {
      if (threadIdx.x < 64) {
        const Key b = bar(ts);
        if (threadIdx.x == 0) ts.last = b;
      }
      __syncthreads();
    }
    const Key least = kWaves > 1 ? ts.last : bar(ts);
    // The vectors of whoever may hold one of the best are looked through again.
    const bool look = !better(least, most);
    const A enough = value_at_least(least);
    if (look && single >= 0) offer(ts, static_cast<A>(alone), (u32)single, least, enough);
    if (once) {
      if (look) {
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
          const int j = j0 + k * BLOCK + threadIdx.x;
          if (j >= j1) break;
          if (!(largest(v[k]) >= enough)) continue;
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            offer(ts, static_cast<A>(v[k].v[i]), (u32)(vecs.column(j) + i), least, enough);
        }
      }
    } else {
      // They are not at hand any more: all lanes of a wave share those of its
      // threads (216 rows of 155176 float32, 5 of them: 35 us; 38 with every thread
      // after its own, 50 of them one by one).
      const int lane = threadIdx.x & 63;
      const unsigned long long lookers = __ballot(look), below = (1ull << lane) - 1;
      const int count = __popcll(lookers);
      // lane r is told the r-th of them
      const int to = look ? __popcll(lookers & below) : count + __popcll(~lookers & below);
      const int list = __builtin_amdgcn_ds_permute(to * 4, (int)threadIdx.x);
      const u32 trips = (j1 - j0 + BLOCK - 1) / BLOCK, items = count * trips;
      constexpr int kAgain = 4;
      for (u32 base = 0; base < items; base += 64 * kAgain) {
        cupy::Vec<X_T, VEC> again[kAgain];
        int at[kAgain];
#pragma unroll
        for (int k = 0; k < kAgain; ++k) {
          const u32 item = base + k * 64 + lane, who = item / trips;
          at[k] = j0 + (int)(item - who * trips) * BLOCK + cupy::shfl_idx(list, (int)(who & 63));
          if (item >= items || at[k] >= j1) at[k] = -1;
          again[k] = vecs.load(at[k] < 0 ? j1 - 1 : at[k]);
        }
#pragma unroll
        for (int k = 0; k < kAgain; ++k) {
          if (at[k] < 0 || !(largest(again[k]) >= enough)) continue;
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            offer(ts, static_cast<A>(again[k].v[i]), (u32)(vecs.column(at[k]) + i), least, enough);
        }
      }
    }
    __syncthreads();
    const u32 found = ts.n;
    if (found <= kMost) {
      put_ranked(ts, found, put);
    } else {
      // More than can be ranked (the best lie in the vectors of a few threads):
      // one pass over the row per place, each for the best behind the last.
      bool first = true;
      for (int rank = 0; rank < TOP; ++rank) {
        __syncthreads();
        const Key last = ts.last;
        Key b = no_key(0);
        if (!is_none(other) && (first || better(last, other))) b = other;
        for (int j = j0 + threadIdx.x; j < j1; j += BLOCK) {
          const cupy::Vec<X_T, VEC> w = vecs.load(j);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const A value = static_cast<A>(w.v[i]);
            const Key k = key_at(w, j, i, vecs);
            if (value == value && (first || better(last, k)) && better(k, b)) b = k;
          }
        }
        first = false;
        b = cupy::group_allreduce<64>(b, BestKey());
        if ((threadIdx.x & 63) == 0) ts.key[threadIdx.x >> 6] = b;
        __syncthreads();
        if (threadIdx.x == 0) {
          for (int q = 1; q < kWaves; ++q) b = BestKey()(b, ts.key[q]);
          ts.last = b;
          put(rank, b);
        }
      }
    }
#endif
#endif
    __syncthreads();
  }
}

// The parts of a row joined: a workgroup per row, at most 64 parts.  A chain of
// waits: all that does not depend on a result is requested at the start (8 rows of
// 64 parts, 20 alternatives: about 5 us).
extern "C" __global__ void __launch_bounds__(256)
cupy_token_log_prob_join(const X_T* logits, const I_T* tokens, A* log_prob, A* lse, A* entropy,
                         A* top, long long* index, const A* runs, const long long rows,
                         const int width, const long long pitch, const int parts,
                         const long long at_keys) {
  Outputs out;
  out.log_prob = log_prob;
  out.lse = lse;
  out.entropy = entropy;
  out.top = top;
  out.index = index;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const long long token = tokens[row];
  const A* from = runs + (row * parts + (lane < parts ? lane : 0)) * 3;
  Run run;
  run.m = from[0];
  run.s = from[1];
  run.u = from[2];
#if TOP > 0
  // (the TOP-th best of the first of every part: at most TOP parts have keys as
  // good, TOP each)
  constexpr int kMost = MAX_TOP * MAX_TOP;
  __shared__ TopState<kMost> ts;
  const Key* keys = reinterpret_cast<const Key*>(runs + at_keys) + row * parts * TOP;
  constexpr int kEach = (64 * TOP + 255) / 256;
  Key mine[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int at = q * 256 + threadIdx.x;
    mine[q] = at < parts * TOP ? keys[at] : no_key(0);
  }
  // Every part's keys are in order: the first few of each are the sample.
  if (threadIdx.x < 64) {
    const int each = 64 / parts < TOP ? 64 / parts : TOP;
    Key k = no_key(lane);
    if (lane < parts * each) {
      k = keys[(lane / each) * TOP + lane % each];
      if (is_none(k)) k = no_key(lane);
    }
    ts.sample[lane] = k;
  }
  if (threadIdx.x == 0) ts.n = 0;
#endif
  const A logit = threadIdx.x == 0 ? logit_of(logits + row * pitch, token, width) : A(0);
  if (lane >= parts) {
    run.m = lowest<X_T>::value();
    run.s = run.u = A(0);
  }
  run = join_lanes<64>(run);     // (by every wave for itself)
  const double tail = run.tail();
  if (threadIdx.x == 0) put_row(out, run, tail, logit, token, row, width);
#if TOP > 0
  __syncthreads();
#if TOP == 1
  if (threadIdx.x < 64) {
    const Key b = cupy::group_allreduce<64>(ts.sample[threadIdx.x], BestKey());
    if (threadIdx.x == 0) put_top(out, run, tail, row, 0, b);
  }
#else
  const Key least = bar(ts);
  const A enough = value_at_least(least);
#pragma unroll
  for (int q = 0; q < kEach; ++q)
    if (!is_none(mine[q])) offer(ts, value_of(mine[q]), column_of(mine[q]), least, enough);
  __syncthreads();
  put_ranked(ts, ts.n,
             [&](int rank, const Key& k) { put_top(out, run, tail, row, rank, k); });
#endif
#endif
}
''')

_GRAD = _oc.Source(_COMMON + r'''
// d x_j = g (delta_jt - p_j) - gH p_j (log p_j + H).
_CUPY_DEV X_T gradient(X_T logit, A norm, A gain, A gh, A h, bool hit, bool empty) {
  const A lp = static_cast<A>(logit) - norm, p = exp2_(lp * A(LOG2E));
#ifdef ENTROPY
  // (p = 0 long before log p is at -30000: kept there, so that the product with a
  // large gradient is finite and 0)
  A r = -p * cupy::fma_(gh, max_(lp, A(-30000)) + h, gain);
#else
  A r = -p * gain;
#endif
  if (hit) r += gain;
  return static_cast<X_T>(empty ? A(0) : r);
}

// Bound by memory: read once, written once.  Vectors start on cache lines, so that
// waves store whole ones (8192 x 50257 float16 with entropy: 267 us; 289 from
// 16-byte borders).
extern "C" __global__ void __launch_bounds__(BLOCK)
cupy_token_log_prob_grad(const A* g, const X_T* logits, const I_T* tokens, const A* lse,
                         const A* entropy, const A* entropy_grad, X_T* out,
                         const long long rows, const int width, const long long pitch,
                         const long long po, const int blocks) {
  for (long long w = blockIdx.x; w < rows * blocks; w += gridDim.x) {
    const long long row = w / blocks;
    const int block = (int)(w - row * blocks);
    const X_T* x = logits + row * pitch;
    const RowVecs<128> vecs(x, width);
    X_T* to = out + row * po;
    const A norm = lse[row];
    const long long token = tokens[row];
    const bool met = token >= 0 && token < width;
    const int target = met ? (int)token : -1;
    const A gain = met ? g[row] : A(0);
    A gh = A(0), h = A(0);
#ifdef ENTROPY
    gh = entropy_grad[row];
    h = entropy[row];
#endif
    // a row with nothing left has no distribution to change: all -inf, or all the
    // lowest value, where lse has no digits left to tell how many they are
    const bool empty = norm <= (sizeof(A) == 8 ? A(-1.7976931348623157e308) : A(-3.4028234663852886e38));
    const int base = block * BLOCK * UNROLL + threadIdx.x;
    cupy::Vec<X_T, VEC> v[UNROLL];
    if (vecs.n > 0) {
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        const int j = base + k * BLOCK;
        v[k] = vecs.load(j < vecs.n ? j : vecs.n - 1);
      }
    }
    if (block == 0) {
      // (a workgroup has as many threads as a line has elements)
      const int t = threadIdx.x, behind = width - vecs.tail + t;
      const X_T first = x[t < vecs.head ? t : 0], last = x[t < vecs.tail ? behind : 0];
      if (t < vecs.head) to[t] = gradient(first, norm, gain, gh, h, t == target, empty);
      if (t < vecs.tail) to[behind] = gradient(last, norm, gain, gh, h, behind == target, empty);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int j = base + k * BLOCK;
      if (j >= vecs.n) break;
      const int hit = target - vecs.column(j);
      cupy::Vec<X_T, VEC> d;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        d.v[e] = gradient(v[k].v[e], norm, gain, gh, h, hit == e && met, empty);
      cupy::store_vec<X_T, VEC, NT_OUT>(to + vecs.column(j), d);
    }
  }
}
''')

_plans = {}
_plans_grad = {}


def _check_logits(logits, tokens):
    _oc.check_float(logits, 'logits')
    if logits.ndim == 0:
        raise ValueError('logits must have at least one dimension')
    if tokens._shape != logits._shape[:-1]:
        raise ValueError('tokens has the shape %r, logits the shape %r: one token per row is '
                         'expected' % (tokens._shape, logits._shape))
    width = logits._shape[-1]
    if width >= 1 << 31:
        raise ValueError('rows of 2**31 elements and more are not supported')
    if width == 0 and tokens.size:
        raise ValueError('zero-size rows of logits have no distribution')
    return width


def token_log_prob(logits, tokens, *, entropy=False, top=0, out=None):
    """Log probability of one token per row of logits.

    Args:
        logits (cupy.ndarray): float16, float32 or float64, ``(..., n)``;
            elements of -inf are ruled out.
        tokens: integers of shape ``logits.shape[:-1]``.  A token outside
            ``[0, n)`` marks a row without a target: its log probability is 0.
        entropy (bool): also the entropy of every row's distribution.
        top (int): also the ``top`` likeliest tokens of every row (at most 32
            and ``n``) and their log probabilities, likeliest first; of equally
            likely ones the lower token comes first.
        out (TokenLogProb): arrays that receive the results.

    Sums are held and joined in 32 bits (64 for float64), what follows from a row's
    sums is computed in 64.  They are grouped by 16-byte vectors: rows that start
    elsewhere modulo 16 bytes may differ in the last bits.  A row whose elements are
    all -inf has log probabilities of -inf and the entropy 0; a row with a NaN or
    +inf has NaN for all of them and -1 for its likeliest tokens (a token out of range
    has the log probability 0 there too).

    Returns:
        TokenLogProb: ``log_prob``, ``lse`` (the logarithm of the sum of
        exponentials, which the gradient takes), ``entropy``, ``top_log_prob``
        and ``top_token``; float32 (float64 for float64) and int64.
    """
    entropy, top = bool(entropy), operator.index(top)
    arrays = [logits, tokens]
    given = None
    if out is not None:
        if type(out) is not TokenLogProb:
            raise TypeError('out must be a TokenLogProb')
        arrays += [a for a in out if a is not None]
        given = (out.entropy is None, out.top_log_prob is None, out.top_token is None)
    result, key = _oc.replay(_plans, arrays, (entropy, top, given))
    if result is not _oc._NOTHING:
        return _named(result, entropy, top)
    as_given, tokens = tokens, _oc.index_array(tokens, 'tokens')
    if as_given is not tokens:
        key, arrays[1] = None, tokens
    width = _check_logits(logits, tokens)
    if not 0 <= top <= min(MAX_TOP, width):
        raise ValueError('top must be between 0 and %d, got %d' % (min(MAX_TOP, width), top))
    acc = _oc.acc_dtype(logits.dtype)
    lead = logits._shape[:-1]
    specs = [(lead, acc, 'log_prob'), (lead, acc, 'lse')]
    if entropy:
        specs.append((lead, acc, 'entropy'))
    if top:
        specs.append((lead + (top,), acc, 'top_log_prob'))
        specs.append((lead + (top,), numpy.dtype(numpy.int64), 'top_token'))
    if out is not None:
        asked = {name for _, _, name in specs}
        for name, a in zip(out._fields, out):
            if (a is None) == (name in asked):
                raise ValueError('out.%s is %s' % (
                    name, 'missing' if a is None else 'given, but was not asked for'))
        for shape, dt, name in specs:
            _oc.check_out(getattr(out, name), shape, dt, 'out.' + name)
    call = _oc.Call(_plans, key, arrays, 2)
    if out is None:
        at = [call.allocate(shape, dt) for shape, dt, _ in specs]
    else:
        at = list(range(2, 2 + len(specs)))
    ret = tuple(at)
    rows = tokens.size
    if rows == 0:
        call.key = None
        call.begin()
        return _named(call.finish(ret), entropy, top)
    call.convert(1, _oc.as_index(call.refs[1]))
    pitch = call.rows(0)
    for i in at:
        call.dense(i)
    call.begin()
    vec = 16 // logits.dtype.itemsize
    block, unroll, parts = _geometry(rows, max(1, width // vec), top)
    nt_in = _oc.stream_hints(logits.nbytes, 0)[0] and not top
    defines = dict(X_T=logits.dtype, I_T=call.refs[1].dtype, BLOCK=block, UNROLL=unroll, VEC=vec,
                   TOP=top, MAX_TOP=MAX_TOP, SMALL_KEYS=int(acc == numpy.float32), NT_IN=nt_in, NT_OUT=False)
    if entropy:
        defines['ENTROPY'] = 1
    slots = [Ref(i) for i in at[:2]]
    slots.append(Ref(at[2]) if entropy else 0)
    slots += [Ref(at[-2]), Ref(at[-1])] if top else [0, 0]
    at_keys = -(-rows * parts * 3 // 4) * 4          # (keys of 8 or 16 bytes)
    if parts > 1:
        i_t = call.temp((at_keys + rows * parts * top * 2) * acc.itemsize)
        slots.append(Ref(i_t))
    else:
        slots.append(0)
    fn = _SOURCE.function('cupy_token_log_prob', **defines)
    grid = min(rows * parts, 0xffffffff // block)
    values = slots + [rows, width, pitch, parts, at_keys]
    call.launch(fn, (grid, 1, 1), block, 'PPPPPPPPqiqiq', Ref(0), Ref(1), *values)
    if parts > 1:
        fn = _SOURCE.function('cupy_token_log_prob_join', **defines)
        call.launch(fn, (rows, 1, 1), 256, 'PPPPPPPPqiqiq', Ref(0), Ref(1), *values)
    return _named(call.finish(ret), entropy, top)


def _geometry(rows, vecs, top):
    """(threads of a workgroup, vectors a thread requests at a time, parts of a row)"""
    units = _oc.compute_units()
    block, parts = 256, 1
    if rows < units * 3 // 8 and vecs > 14336:
        # Long rows, too few to fill the device, are cut into parts; a second
        # launch joins them, which costs about 5 us (with 5 alternatives: 64 rows of
        # 128000 float16: 13.6 us in parts, 14.0 in one launch; 64 of 200000 float32:
        # 18.0 and 21.2; 8 of 131072 float32: 12.8 and 14.7; but 100 of 64000 float32:
        # 14.4 and 11.4, 32 of 50257: 11.7 and 10.1; with the entropy alone: 12.2 and
        # 12.1, 13.6 and 19.7, 11.8 and 12.7, 12.0 and 9.1, 12.3 and 7.4).
        parts = min(64, max(1, 4 * units // rows), -(-vecs // (2 * block)))
    elif rows <= units and vecs > 2048:
        # (190 rows of 100000 float16 with entropy: 11.0 us; 11.8 with 512 threads to a
        # row, 15.6 with 256; with 5 alternatives: 13.6, 14.0, 18.0)
        block = 1024
    elif rows < 4 * units:
        # (300 rows of 100000 float16 with entropy: 17.7 us with 512 threads to a row,
        # 19.8 with 256, 19.5 with 1024; with 5 alternatives: 19.8, 21.3, 24.8; 1000 rows
        # of 16000 float16: 9.9 and 9.3 with entropy, 15.7 and 12.5 with alternatives)
        block = 512 if vecs > 2048 else 256
    elif vecs <= 512 or (top > 1 and vecs <= 1024):
        # Short rows: one wave to each, whose reductions meet no barrier (16384
        # rows of 1500 float16 with entropy: 15.8 us; 20.5 with two waves, 27.8 with
        # four).  What is done for alternatives is done by every wave, so that fewer are
        # best there (8000 rows of 8000 float16, 5 of them: 35.3 us; 40.2 with two waves,
        # 52.2 with four).
        block = 64
    elif top > 1 and vecs <= 2048:
        # (4000 rows of 8000 float32, 5 of them: 32.2 us; 32.0 with one wave, 37.3 with
        # four)
        block = 128
    # Long ones: four waves, so that a unit holds eight rows (8192 rows of 50257
    # float16 with entropy: 131 us; 142 with eight waves, 197 with sixteen).
    return block, 4, parts


def _named(results, entropy, top):
    results = iter(results)
    return TokenLogProb(next(results), next(results), next(results) if entropy else None,
                        *((next(results), next(results)) if top else (None, None)))


def token_log_prob_grad(grad, logits, tokens, lse, *, entropy=None, entropy_grad=None, out=None):
    """Gradient of :func:`token_log_prob` with respect to the logits.

    ``out[j] = grad * ((j == token) - p[j])``, and with ``entropy_grad`` also
    ``- entropy_grad * p[j] * (log(p[j]) + entropy)``, ``p = exp(logits - lse)``.
    A row whose token is out of range has no part in the first term; a row
    whose elements are all -inf, or the lowest float32 or float64 in logits of these
    types, has the gradient 0.  ``lse`` is taken as it is rounded: float32 logits of a magnitude ``m`` have ``p`` to ``m * 2**-24``.

    Args:
        grad (cupy.ndarray): gradient of ``log_prob``, one per row.
        logits, tokens: as in the forward call.
        lse (cupy.ndarray): ``lse`` of the forward call.
        entropy, entropy_grad (cupy.ndarray): ``entropy`` of the forward call
            and its gradient (both or neither).
        out (cupy.ndarray): receives the gradient, of the shape and type of
            ``logits``; may be ``logits`` itself.
    """
    arrays = [grad, logits, tokens, lse]
    if entropy is not None:
        arrays.append(entropy)
    if entropy_grad is not None:
        arrays.append(entropy_grad)
    if out is not None:
        arrays.append(out)
    with_entropy = entropy_grad is not None
    result, key = _oc.replay(
        _plans_grad, arrays, (entropy is None, entropy_grad is None, out is None))
    if result is not _oc._NOTHING:
        return result
    if (entropy is None) != (entropy_grad is None):
        raise ValueError('entropy and entropy_grad are given together or not at all')
    given, tokens = tokens, _oc.index_array(tokens, 'tokens')
    if given is not tokens:
        key, arrays[2] = None, tokens
    width = _check_logits(logits, tokens)
    acc = _oc.acc_dtype(logits.dtype)
    per_row = [(0, 'grad'), (3, 'lse')]
    if with_entropy:
        per_row += [(4, 'entropy'), (5, 'entropy_grad')]
    for i, name in per_row:
        _oc.check_float(arrays[i], name)
        if arrays[i]._shape != tokens._shape:
            raise ValueError('%s has the wrong shape: %r, expected %r'
                             % (name, arrays[i]._shape, tokens._shape))
    if out is not None:
        _oc.check_out(out, logits._shape, logits.dtype)
    n_in = 6 if with_entropy else 4
    call = _oc.Call(_plans_grad, key, arrays, n_in, [(1, n_in)])
    i_out = n_in if out is not None else call.allocate(logits._shape, logits.dtype)
    if logits.size == 0:
        call.key = None
        call.begin()
        return call.finish(i_out)
    for i, _ in per_row:
        if call.refs[i].dtype != acc:
            call.convert(i, call.refs[i].astype(acc))
        call.dense(i)
    call.convert(2, _oc.as_index(call.refs[2]))
    pitch, po = call.rows(1), call.rows(i_out)
    call.begin()
    rows = tokens.size
    vec = 16 // logits.dtype.itemsize
    vecs = max(1, width // vec)
    # four vectors a thread; short rows: as many waves as take a vector per lane
    unroll = 4 if vecs > 1024 else 2 if vecs > 256 else 1
    block = min(256, -(-vecs // 64) * 64)
    blocks = -(-vecs // (block * unroll))
    nt_in, nt_out = _oc.stream_hints(logits.nbytes, logits.nbytes)
    defines = dict(X_T=logits.dtype, I_T=call.refs[2].dtype, BLOCK=block, UNROLL=unroll, VEC=vec,
                   TOP=0, NT_IN=nt_in, NT_OUT=nt_out)
    if with_entropy:
        defines['ENTROPY'] = 1
    fn = _GRAD.function('cupy_token_log_prob_grad', **defines)
    call.launch(fn, (min(rows * blocks, 0xffffffff // block), 1, 1), block, 'PPPPPPPqiqqi',
                Ref(0), Ref(1), Ref(2), Ref(3), Ref(4) if with_entropy else 0,
                Ref(5) if with_entropy else 0, Ref(i_out), rows, width, pitch, po, blocks)
    return call.finish(i_out)
