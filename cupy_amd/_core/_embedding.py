"""Lookup of table rows with scaling, and its gradient summed by sorted tokens.

``embedding`` gathers rows; ``embedding_grad`` adds the rows of a gradient that
belong to the same row of the table.  Where ``ufunc.at`` would add atomically,
in an order that changes from call to call, the gradient is summed in the order
of the positions: the pairs (token, position) are sorted (a stable radix sort
with the positions as its payload), cut into chunks of equal length whatever
the tokens are, and every chunk sums its runs of equal tokens in registers.
Runs that cross the border of a chunk leave partial sums that a last kernel
joins, in order.  Few tokens need no sort: each is compared with all others.
The reference scatters such gradients atomically
(cupy/_core/_routines_indexing.pyx:899-1120 ``_scatter_op``).
"""
import math
import operator

import numpy

from cupy_amd import _rt
from cupy_amd._core import _op_calls as _oc
from cupy_amd._core._op_calls import Ref

_LOOKUP = _oc.Source(r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<X_T>::type A;

// LANES lanes share a row, each moves ITEMS vectors, all requested before the
// first is stored; blockIdx.y walks the rest of a wide row.  Bound by memory:
// nothing is computed but the product with the scale (none at all at 1, so
// that NaN payloads stay).  16384 rows of 2048 float32: 37 us, 7.2 TB/s counting
// every row once, of which the cache gives the repeated ones.
extern "C" __global__ void __launch_bounds__(256)
cupy_embedding(const X_T* table, const I_T* ids, X_T* out, const long long n, const int width,
               const long long rows, const long long pt, const long long po, const double scale) {
  const int lane = threadIdx.x % LANES;
  const long long step = (long long)gridDim.x * (256 / LANES);
  for (long long t = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; t < n; t += step) {
    const long long id = ids[t];
    const bool met = id >= 0 && id < rows;
    const X_T* row = table + (met ? id : 0) * pt;      // (the table has a row)
    cupy::Vec<X_T, VEC> v[ITEMS];
    int c[ITEMS];
    // A vector over the end of the row moves back to end with it: what it shares
    // with its neighbour is stored twice.  Nothing stands between the requests.
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      c[k] = ((blockIdx.y * ITEMS + k) * LANES + lane) * VEC;
      const int at = TINY ? 0 : c[k] + VEC <= width ? c[k] : width - VEC;
      v[k] = TINY ? cupy::load_part<X_T, VEC>(row, width) : cupy::load_vec<X_T, VEC>(row + at);
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (c[k] >= width) break;
      const int at = TINY ? 0 : c[k] + VEC <= width ? c[k] : width - VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
#ifdef SCALE
        v[k].v[e] = static_cast<X_T>(static_cast<A>(v[k].v[e]) * static_cast<A>(scale));
#endif
        if (!met) v[k].v[e] = static_cast<X_T>(0.0f);
      }
      if (TINY) cupy::store_part<X_T, VEC>(out + t * po, v[k], width);
      else cupy::store_vec<X_T, VEC, NT_OUT>(out + t * po + at, v[k]);
    }
  }
}
''')

# -- the sort ---------------------------------------------------------------------------
# Up to _RANKED pairs whose token and position fit one word are put in order by
# counting, for each, the pairs before it.  More of them are sorted digit by
# digit, in two launches per digit: workgroups of 1024 threads count the digits
# of their tiles, then every pair moves to its place: behind the smaller digits
# of all tiles, the equal ones of earlier tiles, and the equal ones before it in
# its own.  Equal digits keep their order, so the sort is stable and its result
# does not depend on the order in which anything runs.
# The result is cleared by further workgroups of the same launches, an equal
# share of its rows in each: the sort keeps few units busy and hides behind them.

_GRAD = _oc.Source(r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<G_T>::type A;
typedef unsigned int u32;

constexpr int kThreads = 1024;
constexpr int kWaves = 16;
constexpr int kBins = 512;
constexpr int kTile = ROUNDS * kThreads;

struct Digits {
  // per wave: how many, then the first place inside the digit (at most kTile)
  unsigned short count[kWaves][kBins];
  u32 first[kBins];           // first place of a digit
  u32 wave_total[kWaves];
};

_CUPY_DEV u32 digit_of(u32 key, int shift, int bits) { return (key >> shift) & ((1u << bits) - 1); }

// The place of every key among the tile's keys of the same digit within the
// wave, and count[][] filled in.
_CUPY_DEV void count_digits(Digits& s, const u32 (&key)[ROUNDS], u32 (&place)[ROUNDS],
                            int shift, int bits) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < kWaves * kBins; i += kThreads) s.count[i / kBins][i % kBins] = 0;
  __syncthreads();
  volatile unsigned short* mine = s.count[wave];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const u32 d = digit_of(key[r], shift, bits);
    unsigned long long same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const unsigned long long set = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? set : ~set;
    }
    const u32 before = __popcll(same & ((1ull << lane) - 1));
    // (every lane reads the count of its digit before the first of the lanes
    // that share it raises it: LDS accesses of a wave happen in program order)
    const u32 had = mine[d];
    place[r] = had + before;
    __builtin_amdgcn_wave_barrier();
    if (before == 0) mine[d] = static_cast<unsigned short>(had + __popcll(same));
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
}

// count[w][d] becomes the number of d's in the waves before w.
_CUPY_DEV void sum_waves(Digits& s) {
  if (threadIdx.x < kBins) {
    u32 c[kWaves], total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) c[w] = s.count[w][threadIdx.x];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      s.count[w][threadIdx.x] = static_cast<unsigned short>(total);
      total += c[w];
    }
  }
}

// Exclusive sums over the first kBins threads' values, plus `offset`, to first[].
_CUPY_DEV void first_places(Digits& s, u32 value, u32 offset) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u32 v = value;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u32 o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  if (lane == 63) s.wave_total[wave] = v;
  __syncthreads();
  u32 base = 0;
  for (int w = 0; w < wave; ++w) base += s.wave_total[w];
  if (threadIdx.x < kBins) s.first[threadIdx.x] = base + v - value + offset;
  __syncthreads();
}

_CUPY_DEV u32 key_of(long long id, u32 rows) {
  return id >= 0 && id < (long long)rows ? (u32)id : rows;    // no row: behind all rows
}

// Zeros to the rows [r0, r1) of the result, by the workgroups from `first_block`
// on, of which one to a unit, and four of its waves, store fastest (537 MB: 84 us;
// all sixteen waves 94, of two workgroups 111, of four 126).
_CUPY_DEV void clear_rows(O_T* out, u32 r0, u32 r1, int width, long long po, int first_block) {
  constexpr int kStoring = 256;
  if (threadIdx.x >= kStoring) return;
  const long long blocks = gridDim.x - first_block, block = blockIdx.x - first_block;
  cupy::Vec<O_T, FILL_VEC> zero;
#pragma unroll
  for (int e = 0; e < FILL_VEC; ++e) zero.v[e] = static_cast<O_T>(0.0f);
  if (po == width) {
    // stored one after the other: one piece
    out += (long long)r0 * width;
    const long long length = (long long)(r1 - r0) * width, vecs = length / FILL_VEC;
    const long long me = block * kStoring + threadIdx.x;
    for (long long i = me; i < vecs; i += blocks * kStoring)
      cupy::store_vec<O_T, FILL_VEC, NT_OUT>(out + i * FILL_VEC, zero);
    if (me < length - vecs * FILL_VEC) out[vecs * FILL_VEC + me] = zero.v[0];
  } else {
    for (long long r = r0 + block; r < r1; r += blocks)
      for (int c = threadIdx.x; c < width; c += kStoring) out[r * po + c] = zero.v[0];
  }
}

// Few tokens: the place of a pair is the number of pairs before it, counted by
// comparing it with all of them: the work grows with the square, but is spread
// over the whole device and takes one short step instead of a chain of them.
// A pair is one word, its token above its position.  16 * EACH pairs by 64
// slices of all pairs to a workgroup.  4001 pairs: 6.3 us, 16 MB cleared beside it.
extern "C" __global__ void __launch_bounds__(kThreads)
cupy_embedding_rank(const I_T* ids, u32* pairs, O_T* out, const int n, const u32 rows,
                    const int width, const long long po, const int position_bits,
                    const int blocks) {
  constexpr int kLoads = EACH * 4;                   // 4096 * EACH pairs at most
  __shared__ u32 all[kLoads * kThreads];
  __shared__ u32 count[kWaves][16 * EACH];
  if ((int)blockIdx.x >= blocks) {
    clear_rows(out, 0, rows, width, po, blocks);
    return;
  }
  long long id[kLoads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int i = k * kThreads + (int)threadIdx.x;
    id[k] = ids[i < n ? i : n - 1];
  }
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int i = k * kThreads + (int)threadIdx.x;
    all[i] = i < n ? key_of(id[k], rows) << position_bits | i : 0xffffffffu;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slice = (n + 255) / 256;                 // in 16-byte words
  const uint4* from = reinterpret_cast<const uint4*>(all) + (wave * 4 + (lane >> 4)) * slice;
  u32 me[EACH], before[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int mine = (blockIdx.x * EACH + e) * 16 + (lane & 15);
    me[e] = mine < n ? all[mine] : 0u;
    before[e] = 0;
  }
#pragma unroll 2
  for (int i = 0; i < slice; ++i) {
    const uint4 k = from[i];
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      before[e] += (k.x < me[e]) + (k.y < me[e]) + (k.z < me[e]) + (k.w < me[e]);
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    before[e] += __shfl_xor(before[e], 16, 64);
    before[e] += __shfl_xor(before[e], 32, 64);
    if (lane < 16) count[wave][e * 16 + lane] = before[e];
  }
  __syncthreads();
  const int mine = blockIdx.x * EACH * 16 + (int)threadIdx.x;
  if (threadIdx.x < 16 * EACH && mine < n) {
    u32 at = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) at += count[w][threadIdx.x];
    pairs[at] = all[mine] >> position_bits;
    pairs[n + at] = mine;
  }
}

// Keys and positions of a pass over many tiles: the first pass reads the tokens.
_CUPY_DEV void load_tile(const I_T* ids, const u32* from, u32 (&key)[ROUNDS], u32 (&pos)[ROUNDS],
                         long long n, u32 rows, bool first) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const long long i = (long long)blockIdx.x * kTile + (wave * ROUNDS + r) * 64 + lane;
    key[r] = 0xffffffffu;
    pos[r] = (u32)i;
    if (i < n) {
      key[r] = first ? key_of(ids[i], rows) : from[i];
      if (!first) pos[r] = from[n + i];
    }
  }
}

// counts[tile][digit]; the workgroups behind the tiles clear rows of the result,
// which is what it takes (16384 pairs and 134 MB: 21 us, as the next kernel).
extern "C" __global__ void __launch_bounds__(kThreads)
cupy_embedding_count(const I_T* ids, u32* temp, const long long from, const long long at_counts,
                     O_T* out, const long long n, const u32 rows, const int width,
                     const long long po, const int shift, const int bits, const int tiles,
                     const u32 clear0, const u32 clear1) {
  __shared__ u32 count[kBins];
  if ((int)blockIdx.x >= tiles) {
    clear_rows(out, clear0, clear1, width, po, tiles);
    return;
  }
  if (threadIdx.x < kBins) count[threadIdx.x] = 0;
  u32 key[ROUNDS], pos[ROUNDS];
  load_tile(ids, temp + from, key, pos, n, rows, shift == 0);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) atomicAdd(&count[digit_of(key[r], shift, bits)], 1u);
  __syncthreads();
  if (threadIdx.x < kBins)
    temp[at_counts + (long long)blockIdx.x * kBins + threadIdx.x] = count[threadIdx.x];
}

extern "C" __global__ void __launch_bounds__(kThreads)
cupy_embedding_move(const I_T* ids, u32* temp, const long long from, const long long to_at,
                    const long long at_counts, O_T* out, const long long n, const u32 rows,
                    const int width, const long long po, const int shift, const int bits,
                    const int tiles, const u32 clear0, const u32 clear1) {
  __shared__ Digits s;
  if ((int)blockIdx.x >= tiles) {
    clear_rows(out, clear0, clear1, width, po, tiles);
    return;
  }
  u32 key[ROUNDS], pos[ROUNDS], place[ROUNDS];
  load_tile(ids, temp + from, key, pos, n, rows, shift == 0);
  // how many of a digit there are, and how many in the tiles before this one
  u32 all = 0, before = 0;
  if (threadIdx.x < kBins) {
    const u32* c = temp + at_counts + threadIdx.x;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
      const u32 v = c[(long long)t * kBins];
      all += v;
      before += t < (int)blockIdx.x ? v : 0;
    }
  }
  count_digits(s, key, place, shift, bits);
  sum_waves(s);
  first_places(s, all, before);
  u32* to = temp + to_at;
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const u32 d = digit_of(key[r], shift, bits);
    const long long at = (long long)s.first[d] + s.count[wave][d] + place[r];
    // (the filling of the last tile has the largest digit and the last places)
    if (at < n) {
      to[at] = key[r];
      to[n + at] = pos[r];
    }
  }
}
''')

_SUMS = _oc.Source(r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<G_T>::type A;
typedef unsigned int u32;

_CUPY_DEV void put(O_T* out, const A (&sum)[VEC], int have, A scale) {
  cupy::Vec<O_T, VEC> v;
#pragma unroll
  for (int e = 0; e < VEC; ++e) v.v[e] = static_cast<O_T>(sum[e] * scale);
  cupy::store_part<O_T, VEC>(out, v, have);
}

// LANES lanes across the columns; a chunk of `chunk` sorted pairs to each such
// group.  Rows of the gradient are requested UNROLL at a time.
// partial[chunk][0]: the sum of a run that began in an earlier chunk;
// partial[chunk][1]: of one that begins here and goes on behind the chunk.
// Bound by memory, 16384 rows of 2048 float16 into as many of 131072: 18.6 us, 5
// TB/s; small ones by the chain from pair to row (4001 of 509 float32: 5 us).
extern "C" __global__ void __launch_bounds__(256)
cupy_embedding_sums(const G_T* g, u32* temp, O_T* out, const long long at_pairs,
                    const long long at_partial, const long long n, const u32 rows,
                    const int width, const long long pg, const long long po, const int chunk,
                    const int chunks, const double scale_) {
  constexpr int UNROLL = 8;
  const A scale = static_cast<A>(scale_);
  const long long ch = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  int c = (blockIdx.y * LANES + threadIdx.x % LANES) * VEC;
  if (ch >= chunks || c >= width) return;
  // (a vector over the end of the row moves back to end with it: the columns it
  // shares with its neighbour are summed and stored twice, alike)
  if (!TINY && c + VEC > width) c = width - VEC;
  const int have = TINY ? width : VEC;
  const u32* keys = temp + at_pairs;
  const u32* pos = keys + n;
  A* partial = reinterpret_cast<A*>(temp + at_partial);
  const long long t0 = ch * chunk;
  const long long t1 = t0 + chunk < n ? t0 + chunk : n;
  u32 cur = keys[t0];
  const u32 before = keys[t0 > 0 ? t0 - 1 : 0], behind = keys[t1 < n ? t1 : n - 1];
  bool head = t0 > 0 && before == cur;
  u32 key_ahead[UNROLL], at_ahead[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    key_ahead[u] = keys[t0 + u < t1 ? t0 + u : t1 - 1];
    at_ahead[u] = pos[t0 + u < t1 ? t0 + u : t1 - 1];
  }
  if (cur >= rows) return;
  A sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = A(0);
  A* mine = partial + ch * 2 * width + c;
  for (long long t = t0; t < t1; t += UNROLL) {
    u32 key[UNROLL], at[UNROLL];
    cupy::Vec<G_T, VEC> v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      key[u] = key_ahead[u];
      at[u] = at_ahead[u];
    }
    // (positions are in range whatever their token: nothing to wait for)
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      v[u] = TINY ? cupy::load_part<G_T, VEC>(g + (long long)at[u] * pg + c, have)
                  : cupy::load_vec<G_T, VEC>(g + (long long)at[u] * pg + c);
    const long long ahead = t + UNROLL < t1 ? t + UNROLL : t;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      key_ahead[u] = keys[ahead + u < t1 ? ahead + u : t1 - 1];
      at_ahead[u] = pos[ahead + u < t1 ? ahead + u : t1 - 1];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (t + u >= t1) break;
      if (key[u] != cur) {
        if (cur < rows) {
          if (head) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (e < have) mine[e] = sum[e];
          } else {
            put(out + (long long)cur * po + c, sum, have, scale);
          }
        }
        head = false;
        cur = key[u];
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] = A(0);
      }
      if (cur < rows) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] += static_cast<A>(v[u].v[e]);
      }
    }
  }
  if (cur >= rows) return;
  const bool on = t1 < n && behind == cur;
  if (!head && !on) {
    put(out + (long long)cur * po + c, sum, have, scale);
  } else {
    A* to = head ? mine : mine + width;
#pragma unroll
    for (int e = 0; e < VEC; ++e) if (e < have) to[e] = sum[e];
  }
}

// The runs that cross chunks, each by the workgroups of the chunk it begins
// in: 64 lanes of JVEC columns by 4 slices of the chunks it goes on through.  A
// chain of waits: 5.4 us.
extern "C" __global__ void __launch_bounds__(256)
cupy_embedding_join(const u32* temp, O_T* out, const long long at_pairs,
                    const long long at_partial, const long long n, const u32 rows,
                    const int width, const long long po, const int chunk, const int chunks,
                    const double scale) {
  constexpr int JVEC = 16 / sizeof(A);
  __shared__ cupy::Vec<A, JVEC> lds[4][64];
  const u32* keys = temp + at_pairs;
  const A* partial = reinterpret_cast<const A*>(temp + at_partial);
  const long long ch = blockIdx.x;
  const long long t0 = ch * chunk, t1 = t0 + chunk;
  if (t1 >= n) return;
  const u32 cur = keys[t1], last = keys[t1 - 1], before = keys[t0 > 0 ? t0 - 1 : 0];
  const u32 next = ch + 2 < chunks ? keys[t1 + chunk] : rows;
  if (cur >= rows || last != cur) return;
  if (t0 > 0 && before == cur) return;             // it began before this chunk
  // last chunk that begins with `cur`, 256 looked at together
  long long lo = ch + 1;
  if (next == cur) {
    int found;
    do {
      const long long q = lo + 1 + threadIdx.x;
      found = __syncthreads_count(q < chunks && keys[q * chunk] == cur);
      lo += found;
    } while (found == 256);
  }
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int c = (blockIdx.y * 64 + tx) * JVEC;
  const int have = width - c;
  A t[JVEC];
#pragma unroll
  for (int e = 0; e < JVEC; ++e) t[e] = A(0);
  if (have > 0) {
    // (the first one is the sum of the run's beginning, at the end of its chunk)
    for (long long j = ch + ty; j <= lo; j += 16) {
      cupy::Vec<A, JVEC> p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long q = j + 4 * k <= lo ? j + 4 * k : lo;
        p[k] = cupy::load_part<A, JVEC>(partial + (q * 2 + (q == ch)) * width + c, have);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j + 4 * k <= lo)
#pragma unroll
          for (int e = 0; e < JVEC; ++e) t[e] += p[k].v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < JVEC; ++e) lds[ty][tx].v[e] = t[e];
  __syncthreads();
  if (ty == 0 && have > 0) {
    cupy::Vec<O_T, JVEC> r;
#pragma unroll
    for (int e = 0; e < JVEC; ++e)
      r.v[e] = static_cast<O_T>((((lds[0][tx].v[e] + lds[1][tx].v[e]) + lds[2][tx].v[e]) +
                                 lds[3][tx].v[e]) * static_cast<A>(scale));
    cupy::store_part<O_T, JVEC>(out + (long long)cur * po + c, r, have);
  }
}
''')

# -- few tokens ---------------------------------------------------------------------------
# Up to _FEW of them take one launch without a sort.  A workgroup to every
# position (and 64 vectors of columns) compares its token with all others: the
# first position of a token collects the later ones, in order, and sums their
# rows.  Further workgroups clear the rows of the table that no token names,
# which they find by marking those that are named in a bitmap of their share.
# Bound by latency: the tokens, a row, the result are one chain (1011 tokens, 9846
# x 178 float32: 6.5 us, 13.4 with the sort).

_DIRECT = _oc.Source(r'''
#include <cupy/rows.cuh>
typedef cupy::acc_of<G_T>::type A;
typedef unsigned int u32;
typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kIds = FEW / kThreads;             // tokens that a thread looks at
constexpr int kWords = FEW / 64;                 // of 64 positions
constexpr int kSlices = 4;                       // of a long list of positions: a wave each
constexpr int kMany = 8;                         // ... which is of more than so many

// Zeros to the rows [r0, r1), stored one after the other: vectors from the first
// cache line on, the elements before and behind them one by one.
_CUPY_DEV void clear(O_T* out, long long r0, long long r1, int width) {
  constexpr int kLine = 128 / sizeof(O_T);
  const O_T zero = static_cast<O_T>(0.0f);
  O_T* to = out + r0 * width;
  const long long length = (r1 - r0) * width;
  const int phase = (int)((reinterpret_cast<u64>(to) & 127) / sizeof(O_T));
  long long head = phase ? kLine - phase : 0;
  if (head > length) head = length;
  const long long vecs = (length - head) / FILL_VEC;
  cupy::Vec<O_T, FILL_VEC> zeros;
#pragma unroll
  for (int e = 0; e < FILL_VEC; ++e) zeros.v[e] = zero;
  for (long long i = threadIdx.x; i < vecs; i += kThreads)
    cupy::store_vec<O_T, FILL_VEC>(to + head + i * FILL_VEC, zeros);
  const long long behind = head + vecs * FILL_VEC;
  if (threadIdx.x < head) to[threadIdx.x] = zero;
  if (threadIdx.x < length - behind) to[behind + threadIdx.x] = zero;
}

_CUPY_DEV cupy::Vec<G_T, VEC> row_part(const G_T* from, int width) {
  return TINY ? cupy::load_part<G_T, VEC>(from, width) : cupy::load_vec<G_T, VEC>(from);
}

// The rows at the positions list[q0 .. q1 - 1], kAhead requested at a time: one
// alone, or as many as fit, without a question between the requests.
template <int kAhead>
_CUPY_DEV void add_rows(A (&sum)[VEC], const G_T* g, const unsigned short* list, int q0, int q1,
                        int width, long long pg) {
  for (int q = q0; q < q1; q += kAhead) {
    cupy::Vec<G_T, VEC> v[kAhead];
    const int more = q1 - 1 - q;
    v[0] = row_part(g + (long long)list[q] * pg, width);
    if (more > 0) {
#pragma unroll
      for (int u = 1; u < kAhead; ++u)
        v[u] = row_part(g + (long long)list[q + (u < more ? u : more)] * pg, width);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const A term = static_cast<A>(v[u].v[e]);
        sum[e] = u <= more ? sum[e] + term : sum[e];
      }
    }
  }
}

extern "C" __global__ void __launch_bounds__(kThreads)
cupy_embedding_few(const G_T* g, const I_T* ids, O_T* out, const int n, const u32 rows,
                   const int width, const long long pg, const long long po, const double scale_,
                   const int clearing) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long long id[kIds];
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    const int i = k * kThreads + (int)threadIdx.x;
    id[k] = ids[i < n ? i : n - 1];
  }
  if ((int)blockIdx.x < clearing) {
    __shared__ u32 named[64];                    // of the workgroup's rows, 2048 at most
    if (blockIdx.y > 0) return;
    const long long r0 = (long long)rows * blockIdx.x / clearing;
    const long long r1 = (long long)rows * (blockIdx.x + 1) / clearing;
    if (threadIdx.x < 64) named[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kIds; ++k)
      if (id[k] >= r0 && id[k] < r1)
        atomicOr(&named[(id[k] - r0) >> 5], 1u << ((id[k] - r0) & 31));
    __syncthreads();
    const u32 word = named[lane];
    long long from = r0;
    for (u64 words = __ballot(word != 0); words; words &= words - 1) {
      const int j = __ffsll(words) - 1;
      for (u32 bits = (u32)__builtin_amdgcn_readlane(word, j); bits; bits &= bits - 1) {
        const long long row = r0 + j * 32 + __ffs(bits) - 1;
        if (row > from) clear(out, from, row, width);
        from = row + 1;
      }
    }
    if (r1 > from) clear(out, from, r1, width);
    return;
  }
  __shared__ u64 same[kWords];
  __shared__ unsigned short list[FEW];
  __shared__ cupy::Vec<A, VEC> part[kSlices][64];
  const int t = blockIdx.x - clearing;
  const long long token = ids[t];
  if (token < 0 || token >= (long long)rows) return;
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    const u64 found = __ballot(id[k] == token && k * kThreads + (int)threadIdx.x < n);
    if (lane == 0) same[k * (kThreads / 64) + wave] = found;
  }
  __syncthreads();
  int count = 0, ahead[kIds];
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    const u64 m = same[j];
    // (an earlier position of the same token: its workgroup sums)
    if (j * 64 < t && (m & (t - j * 64 < 64 ? (1ull << (t - j * 64)) - 1 : ~0ull))) return;
    if (j % (kThreads / 64) == wave)
      ahead[j / (kThreads / 64)] = count + __popcll(m & ((1ull << lane) - 1));
    count += __popcll(m);
  }
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    const int i = k * kThreads + (int)threadIdx.x;
    if (id[k] == token && i < n) list[ahead[k]] = static_cast<unsigned short>(i);
  }
  __syncthreads();
  // Few positions: one wave.  Many: a quarter of them to each of four, whose sums
  // are added in order.
  const bool many = count > kMany;
  if (!many && wave > 0) return;
  const int share = many ? (count + kSlices - 1) / kSlices : count;
  const int q0 = wave * share, q1 = q0 + share < count ? q0 + share : count;
  int c = (blockIdx.y * 64 + lane) * VEC;
  const bool mine = c < width;
  // (a vector over the end of the row moves back to end with it)
  c = TINY || !mine ? 0 : c + VEC <= width ? c : width - VEC;
  A sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = A(0);
  if (mine) {
    if (many) add_rows<16>(sum, g + c, list, q0, q1, width, pg);
    else add_rows<kMany>(sum, g + c, list, q0, q1, width, pg);
  }
  if (many) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[wave][lane].v[e] = sum[e];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int s = 1; s < kSlices; ++s)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += part[s][lane].v[e];
  }
  if (mine) {
    const A scale = static_cast<A>(scale_);
    cupy::Vec<O_T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = static_cast<O_T>(sum[e] * scale);
    cupy::store_part<O_T, VEC>(out + token * po + c, r, TINY ? width : VEC);
  }
}
''')

# Most tokens that take one launch.  (All of them one and the same are summed by four
# waves: 1024 tokens, 9846 x 178 float32: 19 us, 17 with the sort; 8191 x 1000: 26 and 19.)
_FEW = 1024
# most pairs that are put in order by comparing all of them
_RANKED = 12288

_plans = {}
_plans_grad = {}


def _check_width(width):
    if width >= 1 << 22:       # (a grid's second dimension)
        raise ValueError('rows of 2**22 elements and more are not supported')


def embedding(table, ids, scale=1.0, *, out=None):
    """Rows of a table, scaled: ``out[...] = scale * table[ids[...]]``.

    An id outside ``[0, len(table))`` selects no row: its row of the result is
    zeros (padding may be marked with -1).

    Args:
        table (cupy.ndarray): float16, float32 or float64 matrix.
        ids: integers of any shape.
        scale (float): factor, of 32 bits (64 for float64 tables); the product is
            rounded once.
        out (cupy.ndarray): receives the result, of shape
            ``ids.shape + (table.shape[1],)`` and the table's type.
    """
    scale = float(scale)
    arrays = [table, ids] if out is None else [table, ids, out]
    # (0.0 and -0.0 are one key, but two results)
    result, key = _oc.replay(_plans, arrays, (scale, math.copysign(1.0, scale)))
    if result is not _oc._NOTHING:
        return result
    _oc.check_float(table, 'table')
    if table.ndim != 2:
        raise ValueError('table must have two dimensions, got %d' % table.ndim)
    given, ids = ids, _oc.index_array(ids, 'ids')
    if given is not ids:
        key, arrays[1] = None, ids
    rows, width = table._shape
    shape = ids._shape + (width,)
    _check_width(width)
    if out is not None:
        _oc.check_out(out, shape, table.dtype)
    call = _oc.Call(_plans, key, arrays, 2)
    i_out = 2 if out is not None else call.allocate(shape, table.dtype)
    n = ids.size
    if n == 0 or width == 0 or rows == 0:
        # (the kernel reads some row for every id: without rows it is not run)
        call.key = None
        if call.refs[i_out].size:
            call.refs[i_out].fill(0)
        call.begin()
        return call.finish(i_out)
    call.convert(1, _oc.as_index(call.refs[1]))
    pt, po = call.rows(0), call.rows(i_out)
    call.begin()
    vec = 16 // table.dtype.itemsize
    vecs = -(-width // vec)
    lanes = min(256, max(4, _oc.clp2(vecs)))
    # Few rows: a vector per lane and the row over more workgroups, so that all
    # of it is requested at once.
    items = 1 if n * vecs < _oc.compute_units() * 2048 else min(4, -(-vecs // lanes))
    grid_y = -(-vecs // (lanes * items))
    per = 256 // lanes
    grid_x = min(-(-n // per), (1 << 24) - 1)
    nt_out = _oc.stream_hints(n * width * table.dtype.itemsize, n * width * table.dtype.itemsize)[1]
    defines = dict(X_T=table.dtype, I_T=call.refs[1].dtype, LANES=lanes, ITEMS=items, VEC=vec,
                   TINY=width < vec, NT_OUT=nt_out)
    if scale != 1.0:
        defines['SCALE'] = 1
    fn = _LOOKUP.function('cupy_embedding', **defines)
    call.launch(fn, (grid_x, grid_y, 1), 256, 'PPPqiqqqd', Ref(0), Ref(1), Ref(i_out), n, width,
                rows, pt, po, scale)
    return call.finish(i_out)


def _chunk(n, pairs, partial, groups, across):
    """Sorted pairs that one group of lanes sums: of n, which take ``pairs`` bytes of
    the temporary beside ``partial`` for each chunk's sums; a workgroup takes
    ``groups`` chunks, ``across`` workgroups the columns."""
    # long enough that few runs cross the borders, short enough that there are some
    # per compute unit
    chunk = min(128, max(8, _oc.clp2(n // 512)))
    # ... and so long that ``static_scratch`` holds the temporary, where that leaves
    # sixteen workgroups to a unit (with eight, 262144 tokens of 4096 float16 take 619 us,
    # 603 with twice as many)
    longer = chunk
    while pairs + -(-n // longer) * partial > _rt.RT_SCRATCH_MAX_BYTES and longer < n:
        longer *= 2
    if -(-(-(-n // longer)) // groups) * across >= 16 * _oc.compute_units():
        chunk = longer
    return chunk


def embedding_grad(grad, ids, num_rows, scale=1.0, *, dtype=None, out=None):
    """Gradient of :func:`embedding` with respect to its table.

    ``out[v] = scale * (sum of grad[t] over all t with ids[t] == v)``; rows
    that no id selects are zeros, ids outside ``[0, num_rows)`` have no part.
    The sums are held in 32 bits (64 for float64), their order follows from the
    sizes, the ids and whether the rows of the result are stored one after the
    other: repeated calls give the same bits.  Under ``cuda.memory.static_scratch``
    about 8 million ids can be taken (16 bytes for each, and the partial sums).

    Args:
        grad (cupy.ndarray): gradient of the looked up rows, of shape
            ``ids.shape + (width,)``; float16, float32 or float64.
        ids: integers, as in the forward call.
        num_rows (int): rows of the table.
        scale (float): as in the forward call.
        dtype: type of the result; the gradient's (default), or float32 with
            float16.
        out (cupy.ndarray): receives the result, ``(num_rows, width)``; not
            both ``out`` and ``dtype``.
    """
    scale = float(scale)
    num_rows = operator.index(num_rows)
    if dtype is not None:
        if out is not None:
            raise TypeError('embedding_grad() takes `out` or `dtype`, but both were provided.')
        dtype = numpy.dtype(dtype)
    arrays = [grad, ids] if out is None else [grad, ids, out]
    result, key = _oc.replay(
        _plans_grad, arrays, (scale, math.copysign(1.0, scale), num_rows, dtype))
    if result is not _oc._NOTHING:
        return result
    _oc.check_float(grad, 'grad')
    given, ids = ids, _oc.index_array(ids, 'ids')
    if given is not ids:
        key, arrays[1] = None, ids
    if grad.ndim != ids.ndim + 1 or grad._shape[:-1] != ids._shape:
        raise ValueError('grad has the shape %r, ids the shape %r: one row per id is expected'
                         % (grad._shape, ids._shape))
    if not 0 <= num_rows < (1 << 31) - 1:
        raise ValueError('num_rows must be at least 0 and below 2**31 - 1')
    width = grad._shape[-1]
    n = ids.size
    _check_width(width)
    if n >= 1 << 30:
        raise ValueError('2**30 ids and more are not supported')
    if out is not None:
        _oc.check_array(out, 'out')
        dt = out.dtype
    else:
        dt = grad.dtype if dtype is None else dtype
    if dt != grad.dtype and not (grad.dtype.char == 'e' and dt.char == 'f'):
        raise TypeError('a gradient of type %s is not summed into %s: its own type, or float32 '
                        'with float16' % (grad.dtype, dt))
    if out is not None:
        _oc.check_out(out, (num_rows, width), dt)
    call = _oc.Call(_plans_grad, key, arrays, 2)
    i_out = 2 if out is not None else call.allocate((num_rows, width), dt)
    if num_rows == 0 or width == 0 or n == 0:
        call.key = None
        if call.refs[i_out].size:
            call.refs[i_out].fill(0)
        call.begin()
        return call.finish(i_out)
    call.convert(1, _oc.as_index(call.refs[1]))
    pg, po = call.rows(0), call.rows(i_out)
    call.begin()
    out_vec = 16 // dt.itemsize
    nt_out = _oc.stream_hints(num_rows * width * dt.itemsize, num_rows * width * dt.itemsize)[1]
    acc = _oc.acc_dtype(grad.dtype).itemsize
    vec = 16 // grad.dtype.itemsize
    units = _oc.compute_units()
    clearing = min(units, num_rows)
    slices = -(-width // (64 * vec))
    # One launch where the comparisons are few (1024 tokens, 8191 x 1009 float32:
    # 11.4 us, 15.8 with the sort; x 2009: 19.7 and 18.9) and the table fits the last
    # cache (131072 x 1024 float16, 268 MB: 50 and 51; x 1000 float32, 524 MB: 99 and 88).
    looked = max(256, _oc.clp2(n))                     # (what every workgroup looks at)
    if (n <= _FEW and n * slices * looked <= 1 << 22 and po == width
            and num_rows * width * dt.itemsize <= 1 << 28 and -(-num_rows // clearing) <= 2048):
        fn = _DIRECT.function('cupy_embedding_few', G_T=grad.dtype, O_T=dt, I_T=call.refs[1].dtype,
                              FEW=looked, VEC=vec, FILL_VEC=out_vec, TINY=width < vec)
        call.launch(fn, (clearing + n, slices, 1), 256, 'PPPiIiqqdi', Ref(0), Ref(1), Ref(i_out), n,
                    num_rows, width, pg, po, scale, clearing)
        return call.finish(i_out)
    fill = min(units, -(-num_rows * width // (out_vec * 256)))

    position_bits = max(1, (n - 1).bit_length())
    rank = n <= _RANKED and num_rows.bit_length() + position_bits <= 32
    each = _oc.clp2(-(-n // 4096)) if rank else 1     # (it holds 4096 * each pairs)
    # tiles of as many rounds as leave 64 of them at most, up to 16
    rounds = 2
    while rounds < 16 and rounds * 1024 * 64 < n:
        rounds *= 2
    tiles = -(-n // (rounds * 1024))
    key_bits = num_rows.bit_length()
    passes = -(-key_bits // 9)
    bits = -(-key_bits // passes)
    # the temporary: sorted pairs (two copies and counts if sorted by digits), partial sums
    words = 2 * n if rank else 4 * n + tiles * 512
    words += words & 1
    lanes = min(256, max(4, _oc.clp2(-(-width // vec))))
    chunk = _chunk(n, words * 4, 2 * width * acc, 256 // lanes, -(-width // (lanes * vec)))
    chunks = -(-n // chunk)
    i_t = call.temp(words * 4 + chunks * 2 * width * acc)
    defines = dict(G_T=grad.dtype, O_T=dt, I_T=call.refs[1].dtype, ROUNDS=rounds,
                   FILL_VEC=out_vec, EACH=each, NT_OUT=nt_out)
    at = 0
    if rank:
        blocks = -(-n // (16 * each))
        fn = _GRAD.function('cupy_embedding_rank', **defines)
        call.launch(fn, (blocks + fill, 1, 1), 1024, 'PPPiIiqii', Ref(1), Ref(i_t), Ref(i_out), n,
                    num_rows, width, po, position_bits, blocks)
    else:
        count = _GRAD.function('cupy_embedding_count', **defines)
        move = _GRAD.function('cupy_embedding_move', **defines)
        at = 2 * n
        cuts = [num_rows * k // (2 * passes) for k in range(2 * passes + 1)]
        for p in range(passes):
            src, at = at, 2 * n - at
            call.launch(count, (tiles + fill, 1, 1), 1024, 'PPqqPqIiqiiiII', Ref(1), Ref(i_t), src,
                        4 * n, Ref(i_out), n, num_rows, width, po, p * bits, bits, tiles,
                        cuts[2 * p], cuts[2 * p + 1])
            call.launch(move, (tiles + fill, 1, 1), 1024, 'PPqqqPqIiqiiiII', Ref(1), Ref(i_t), src,
                        at, 4 * n, Ref(i_out), n, num_rows, width, po, p * bits, bits, tiles,
                        cuts[2 * p + 1], cuts[2 * p + 2])
    defines = dict(G_T=grad.dtype, O_T=dt, LANES=lanes, VEC=vec, TINY=width < vec)
    fn = _SUMS.function('cupy_embedding_sums', **defines)
    call.launch(fn, (-(-chunks // (256 // lanes)), -(-width // (lanes * vec)), 1), 256,
                'PPPqqqIiqqiid', Ref(0), Ref(i_t), Ref(i_out), at, words, n, num_rows, width,
                pg, po, chunk, chunks, scale)
    if chunks > 1:
        fn = _SUMS.function('cupy_embedding_join', **defines)
        call.launch(fn, (chunks, -(-width // (64 * (16 // acc))), 1), 256, 'PPqqqIiqiid', Ref(i_t), Ref(i_out),
                    at, words, n, num_rows, width, po, chunk, chunks, scale)
    return call.finish(i_out)
