// One row of vocabulary logits held by one workgroup: shared by topk.hip, distill.hip and
// filter.hip.
//
// Thread t of NT holds EPT elements in chunks of four neighbours, chunk c at column
// (c * NT + t) * 4, so a wave's load is one contiguous stretch.  EPT = 0 is the row that does not
// fit the registers (V > 65536): every visit reads it again, from the caches after the first.
// Columns from V on hold -inf.
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

template <typename T>
__device__ __forceinline__ void load4(const T* row, int col, int V, float (&v)[4]) {
  if (col + 3 < V) {
    const auto q = *reinterpret_cast<const typename Vec4<T>::type*>(row + col);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)q[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = col + j < V ? (float)row[col + j] : -INFINITY;
  }
}

template <typename T, int NT, int EPT>
struct Row {
  static constexpr int kChunks = EPT / 4;
  float v[kChunks][4];
  const T* row;
  int V;
  __device__ __forceinline__ Row(const T* r, int V_) : row(r), V(V_) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) load4<T>(row, (c * NT + (int)threadIdx.x) * 4, V, v[c]);
  }
  // fn(column of the first, its four values, chunk number)
  template <typename F>
  __device__ __forceinline__ void visit(F&& fn) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) fn((c * NT + (int)threadIdx.x) * 4, v[c], c);
  }
  __device__ __forceinline__ int chunks() const { return kChunks; }
};
template <typename T, int NT>
struct Row<T, NT, 0> {
  const T* row;
  int V;
  __device__ __forceinline__ Row(const T* r, int V_) : row(r), V(V_) {}
  template <typename F>
  __device__ __forceinline__ void visit(F&& fn) {
    const int n = chunks();
    for (int c = 0; c < n; ++c) {
      const int col = (c * NT + (int)threadIdx.x) * 4;
      float v[4];
      load4<T>(row, col, V, v);
      fn(col, v, c);
    }
  }
  __device__ __forceinline__ int chunks() const { return (V + NT * 4 - 1) / (NT * 4); }
};

// ---- reductions over a workgroup of NT threads; `red` holds NT / 64 entries.  Every thread
// gets the result; the trailing barrier frees `red`.
template <int NT, typename T, typename F>
__device__ __forceinline__ T block_reduce(T x, T* red, F&& op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o, 64));
  if constexpr (NT == 64) return x;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = x;
  __syncthreads();
  T r = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r = op(r, red[i]);
  __syncthreads();
  return r;
}
struct AddOp {
  template <typename T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct MaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
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

// Runs fn(NT, EPT) with the workgroup and registers that fit rows of V: one wave up to 1024
// columns (no barriers, and several rows a CU), then more threads before more registers.
#define DCR_ROW_DISPATCH(V, CALL)           \
  do {                                      \
    if ((V) <= 256) { CALL(64, 4); }        \
    else if ((V) <= 1024) { CALL(64, 16); } \
    else if ((V) <= 4096) { CALL(256, 16); } \
    else if ((V) <= 8192) { CALL(256, 32); } \
    else if ((V) <= 32768) { CALL(1024, 32); } \
    else if ((V) <= 65536) { CALL(1024, 64); } \
    else { CALL(1024, 0); }                 \
  } while (0)

}  // namespace dcr
