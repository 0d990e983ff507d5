// One row of vocabulary logits held by one workgroup: shared by topk.hip, distill.hip and
// filter.hip.
//
// The row is cut into chunks of four neighbours for each of NT threads, chunk c of thread t at
// column (c * NT + t) * 4, so a wave's load is one contiguous stretch.  Three holders, one
// interface:
//   Row<T, NT, EPT>   in registers, EPT elements a thread, as stored (bf16 takes half of them)
//   RowLds<T, NT>     in LDS, for kernels with many long visits: their loops stay rolled
//   Row<T, NT, 0>     nowhere: every visit reads the row again, from the caches after the first
// Columns from V on read as -inf.
#pragma once
#include "common.h"
#include "kernels.h"

namespace dcr {

// wide loads and stores at the alignment of one element: rows of an odd width, and padded or
// offset views, start anywhere
typedef float uf32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef bf16 ubf16x4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef uf32x4 type; };
template <> struct Vec4<bf16> { typedef ubf16x4 type; };

// chunk c of this thread: a wave-uniform address and one lane offset for all chunks
template <typename T, int NT>
__device__ __forceinline__ typename Vec4<T>::type load_chunk(const T* row, int c, int V) {
  const T* at = row + c * (NT * 4);
  const unsigned off = threadIdx.x * 4;
  const int left = V - c * (NT * 4);
  typename Vec4<T>::type q;
  if (left >= NT * 4 || (int)off + 3 < left) {
    q = *reinterpret_cast<const typename Vec4<T>::type*>(at + off);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = (int)off + j < left ? at[off + j] : (T)-INFINITY;
  }
  return q;
}
template <typename T>
__device__ __forceinline__ void widen(const typename Vec4<T>::type& q, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (float)q[j];
}
// hides where the values come from, so nothing computed from them is kept for a later visit.
// (Branches around a visit are wave-uniform, and known to be: a value redefined under a divergent
// branch would be held twice.)
__device__ __forceinline__ void forget(uf32x4& q) { asm volatile("" : "+v"(q)); }
__device__ __forceinline__ void forget(ubf16x4& q) { asm volatile("" : "+v"(q)); }

template <typename T, int NT, int EPT>
struct Row {
  static constexpr int kChunks = EPT / 4;
  typename Vec4<T>::type q[kChunks];
  int V;
  __device__ __forceinline__ Row(const T* row, int V_) : V(V_) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) q[c] = load_chunk<T, NT>(row, c, V);
  }
  // fn(column of the first, its four values, chunk number)
  template <typename F>
  __device__ __forceinline__ void visit(F&& fn) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c > 0 && c * NT * 4 >= V) continue;  // nobody's columns (wave-uniform)
      float v[4];
      forget(q[c]);
      widen<T>(q[c], v);
      fn((c * NT + (int)threadIdx.x) * 4, v, c);
      // (long rows: the temporaries of a few chunks at a time)
      if (kChunks >= 16 && c % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
  // sets the values whose bit of drop(column) is set to -inf
  template <typename F>
  __device__ __forceinline__ void erase(F&& drop) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const unsigned bits = drop((c * NT + (int)threadIdx.x) * 4);
      if (bits)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (bits >> j & 1) q[c][j] = (T)-INFINITY;
    }
  }
  // the ones that visit() comes to
  __device__ __forceinline__ int chunks() const { return (V + NT * 4 - 1) / (NT * 4); }
};
template <typename T, int NT>
struct Row<T, NT, 0> {
  static constexpr int kChunks = 0;  // known at run time
  const T* row;
  int V;
  __device__ __forceinline__ Row(const T* r, int V_) : row(r), V(V_) {}
  template <typename F>
  __device__ __forceinline__ void visit(F&& fn) {
    const int n = chunks();
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      const int col = (c * NT + (int)threadIdx.x) * 4;
      float v[4];
      widen<T>(load_chunk<T, NT>(row, c, V), v);
      fn(col, v, c);
    }
  }
  __device__ __forceinline__ int chunks() const { return (V + NT * 4 - 1) / (NT * 4); }
};
template <typename T, int NT>
struct RowLds {  // `lds`: chunks() * NT * 4 elements; each thread reads what it wrote itself
  static constexpr int kChunks = 0;
  typename Vec4<T>::type* own;
  int V;
  __device__ __forceinline__ RowLds(const T* row, int V_, void* lds)
      : own(reinterpret_cast<typename Vec4<T>::type*>(lds) + threadIdx.x), V(V_) {
    const int n = chunks();
#pragma unroll 4
    for (int c = 0; c < n; ++c) own[c * NT] = load_chunk<T, NT>(row, c, V);
  }
  template <typename F>
  __device__ __forceinline__ void visit(F&& fn) {
    const int n = chunks();
#pragma unroll 2
    for (int c = 0; c < n; ++c) {
      float v[4];
      widen<T>(own[c * NT], v);
      fn((c * NT + (int)threadIdx.x) * 4, v, c);
    }
  }
  __device__ __forceinline__ int chunks() const { return (V + NT * 4 - 1) / (NT * 4); }
};

// ---- reductions and scans.  Lanes exchange by DPP moves (a few cycles each; a shuffle goes
// through LDS); all lanes of a wave take part.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp(int old, int x) {
  return __builtin_amdgcn_update_dpp(old, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(dpp<CTRL>(0, __float_as_int(x)));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int x) { return dpp<CTRL>(0, x); }
template <int CTRL>
__device__ __forceinline__ unsigned long long dpp(unsigned long long x) {
  const unsigned lo = (unsigned)dpp<CTRL>(0, (int)(unsigned)x);
  return (unsigned long long)(unsigned)dpp<CTRL>(0, (int)(unsigned)(x >> 32)) << 32 | lo;
}
__device__ __forceinline__ int lane_value(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
__device__ __forceinline__ float lane_value(float x, int l) {
  return __int_as_float(lane_value(__float_as_int(x), l));
}
__device__ __forceinline__ unsigned long long lane_value(unsigned long long x, int l) {
  return (unsigned long long)(unsigned)lane_value((int)(unsigned)(x >> 32), l) << 32 |
         (unsigned)lane_value((int)(unsigned)x, l);
}
// a value that all lanes hold, in a scalar register: branches on it are scalar
template <typename T>
__device__ __forceinline__ T uniform(T x) { return lane_value(x, 0); }
// the wave's result, in every lane: quads, halves and rows of 16 lanes, then the four rows
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T x, F&& op) {
  x = op(x, dpp<0xB1>(x));   // lanes 1 apart
  x = op(x, dpp<0x4E>(x));   // 2 apart
  x = op(x, dpp<0x141>(x));  // the other quad of eight lanes
  x = op(x, dpp<0x140>(x));  // the other eight of the row
  return op(op(lane_value(x, 0), lane_value(x, 16)), op(lane_value(x, 32), lane_value(x, 48)));
}
// inclusive sum over the lanes of a wave: within rows of 16, then the rows in front
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp<0x111>(0, x);
  x += dpp<0x112>(0, x);
  x += dpp<0x114>(0, x);
  x += dpp<0x118>(0, x);
  x += dpp<0x142, 0xa>(0, x);
  x += dpp<0x143, 0xc>(0, x);
  return x;
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

// Over a workgroup of NT threads; `red` holds NT / 64 entries.  Every thread gets the result, and
// `red` is free again.
template <int NT, typename T, typename F>
__device__ __forceinline__ T block_reduce(T x, T* red, F&& op) {
  x = wave_reduce(x, op);
  if constexpr (NT == 64) return x;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  T r = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r = op(r, red[i]);
  __syncthreads();
  return uniform(r);
}
// Several at once, one barrier: x[i] of K values with the same op; `red` holds K * NT / 64.
template <int NT, int K, typename F>
__device__ __forceinline__ void block_reduce_each(float (&x)[K], float* red, F&& op) {
#pragma unroll
  for (int i = 0; i < K; ++i) x[i] = wave_reduce(x[i], op);
  if constexpr (NT == 64) return;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < K; ++i) red[i * (NT / 64) + (threadIdx.x >> 6)] = x[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < K; ++i) {
    x[i] = red[i * (NT / 64)];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) x[i] = op(x[i], red[i * (NT / 64) + w]);
    x[i] = uniform(x[i]);
  }
}
struct AddOp {
  template <typename T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct MaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};
struct MinOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
  __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); }
};

// Order-preserving map between floats (no NaN) and unsigned numbers; -0 counts as +0.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float float_of(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }  // NaN -> -inf

// How many of the row's values satisfy pred(value, column): a ballot per value, so a row of one
// wave counts without any exchange.
template <int NT, typename R, typename P>
__device__ __forceinline__ int count_if(R& row, int* red, P&& pred) {
  int c = 0;
  row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c += (int)__popcll(__ballot(pred(x[j], col + j)));
  });
  if constexpr (NT == 64) return c;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
  __syncthreads();
  c = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) c += red[i];
  __syncthreads();
  return uniform(c);
}

// The place to split a range of keys at: the mean of the two values, which halves the values'
// range (the keys' range holds mostly exponents that no value has), or the mean of the keys
// where that is not between them or has not helped for long.
__device__ __forceinline__ unsigned split_key(unsigned lo, unsigned hi, int round) {
  const unsigned k = key_of(0.5f * float_of(lo) + 0.5f * float_of(hi));
  return round < 24 && k > lo && k < hi ? k : lo + (hi - lo) / 2;
}

// The k-th largest value and the column up to which values equal to it are among the first k.
struct Cut {
  float value;
  int last;
};
// m: the largest value, low: the lowest above -inf.  NaN must read as false in comparisons.
template <int NT, typename R>
__device__ __forceinline__ Cut cut_by_count(R& row, int* red, float m, float low, int k) {
  const int V = row.V;
  unsigned lo = key_of(-INFINITY), hi = key_of(m) + 1;
  int above = 0, have = V;  // count(>= hi) = above < k <= have = count(>= lo)
  if (low > -INFINITY && low <= m) {
    const int c = count_if<NT>(row, red, [&](float x, int) { return x >= low; });
    if (c >= k) lo = key_of(low), have = c; else hi = lo + 1, above = c;
  }
  for (int round = 0; hi - lo > 1 && have != k; ++round) {
    const unsigned mid = split_key(lo, hi, round);
    const float f = float_of(mid);
    const int c = count_if<NT>(row, red, [&](float x, int) { return x >= f; });
    if (c >= k) lo = mid, have = c; else hi = mid, above = c;
  }
  Cut cut{float_of(lo), V - 1};
  if (have != k) {  // more equal values than places: those of the lowest columns
    int a = -1, b = V - 1;
    while (b - a > 1) {
      const int mid = a + (b - a) / 2;
      const int c = count_if<NT>(row, red, [&](float x, int col) {
        return clean(x) == cut.value && col <= mid;
      });
      if (c >= k - above) b = mid; else a = mid;
    }
    cut.last = b;
  }
  return cut;
}

// An entry as one number that orders as the entries do: larger values first, then lower columns.
typedef unsigned long long Entry;
__device__ __forceinline__ Entry entry_of(float x, int col) {
  return (Entry)key_of(x) << 32 | (unsigned)~col;
}
__device__ __forceinline__ float value_of(Entry e) { return float_of((unsigned)(e >> 32)); }
__device__ __forceinline__ int column_of(Entry e) { return (int)~(unsigned)e; }

// Collects the row's entries with pred(value, column) in LDS, in no order; the count goes on past
// `cap`, entries beyond it are not stored.  *count is zero before; a barrier follows.  A row in
// registers is marked first (a bit a value), so a wave asks for its places once; others chunk by
// chunk.
template <int NT, typename R, typename P>
__device__ __forceinline__ void collect(R& row, Entry* list, int* count, int cap, P&& pred) {
  // whether the wave needs places, and the first of this lane's
  auto places = [&](int mine, int& at) {
    const int upto = wave_scan(mine), all = lane_value(upto, 63);
    if (all == 0) return false;
    int base = 0;
    if ((threadIdx.x & 63) == 0) base = atomicAdd(count, all);
    at = uniform(base) + upto - mine;
    return true;
  };
  int at;
  auto put = [&](float x, int col, int at) {
    if (at < cap) list[at] = entry_of(x, col);
  };
  if constexpr (R::kChunks > 0) {
    constexpr int kWords = (R::kChunks + 7) / 8;
    unsigned hit[kWords] = {};
    row.visit([&](int col, float (&x)[4], int c) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        hit[c / 8] |= pred(clean(x[j]), col + j) ? 1u << (c % 8 * 4 + j) : 0u;
    });
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) mine += __popc(hit[i]);
    if (places(mine, at))
      row.visit([&](int col, float (&x)[4], int c) {
        if (hit[c / 8] >> (c % 8 * 4) & 15)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (hit[c / 8] >> (c % 8 * 4 + j) & 1) put(clean(x[j]), col + j, at++);
      });
  } else {
    row.visit([&](int col, float (&x)[4], int) {
      unsigned hit = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) hit |= pred(clean(x[j]), col + j) ? 1u << j : 0u;
      if (places(__popc(hit), at))
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (hit >> j & 1) put(clean(x[j]), col + j, at++);
    });
  }
  __syncthreads();
}

// How many of the c entries in the list, which is 16-byte aligned, come in front of `mine`.
__device__ __forceinline__ int place_of(const Entry* list, int c, Entry mine) {
  struct alignas(16) Two { Entry a, b; };
  const Two* two = reinterpret_cast<const Two*>(list);
  int at = 0;
#pragma unroll 4
  for (int j = 0; j < c / 2; ++j) {
    const Two q = two[j];
    at += (q.a > mine) + (q.b > mine);
  }
  if (c & 1) at += list[c - 1] > mine;
  return at;
}

// A value that at least k of the row reach and, unless many are equal, few more: the row is cut
// into groups of columns, and where k groups have a maximum that high, k values are.  With four
// times k groups or more the overshoot stays small.  -inf where fewer than k groups hold
// anything else.  `gm` holds a value a group (more than one wave).
constexpr int kGroups = 1024;  // for k <= 256
template <int NT, int GROUPS = kGroups, typename R>
__device__ __forceinline__ float reached_by(R& row, float* gm, float* out, int k) {
  constexpr int S = GROUPS / NT;  // groups of one thread's chunks
  float g[S];
#pragma unroll
  for (int i = 0; i < S; ++i) g[i] = -INFINITY;
  row.visit([&](int, float (&x)[4], int c) {
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (c % S == i)
#pragma unroll
        for (int j = 0; j < 4; ++j) g[i] = fmaxf(g[i], x[j]);
  });
  constexpr int kPer = GROUPS / 64;
  float v[kPer];
  if constexpr (NT == 64) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = g[i];
  } else {
#pragma unroll
    for (int i = 0; i < S; ++i) gm[i * NT + threadIdx.x] = g[i];
    __syncthreads();
  }
  if (threadIdx.x < 64) {
    float top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (NT != 64) v[i] = gm[i * 64 + threadIdx.x];
      top = fmaxf(top, v[i]);
      if (v[i] > -INFINITY) low = fminf(low, v[i]);
    }
    top = block_reduce<64>(top, (float*)nullptr, MaxOp());
    low = block_reduce<64>(low, (float*)nullptr, MinOp());
    auto reach = [&](float f) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) c += (int)__popcll(__ballot(v[i] >= f));
      return c;
    };
    float best = -INFINITY;
    if (reach(low) >= k) {
      best = low;
      unsigned lo = key_of(low), hi = key_of(top) + 1;
      int c = GROUPS;
      for (int round = 0; round < 32 && hi - lo > 1 && c > k + k / 8; ++round) {
        const unsigned mid = split_key(lo, hi, round);
        const int q = reach(float_of(mid));
        if (q >= k) lo = mid, c = q, best = float_of(mid); else hi = mid;
      }
    }
    if constexpr (NT == 64) return best;
    if (threadIdx.x == 0) *out = best;
  }
  __syncthreads();
  return uniform(*out);
}

}  // namespace dcr
