// The k largest logits of each row with their indices, and the row's log-sum-exp at a
// temperature: what a teacher records for distillation.  Order: value descending, ties by the
// lowest index; NaN counts as -inf in the order and makes the log-sum-exp NaN.
//
// One workgroup a row.  The row is read once into registers; the k-th largest value is found by
// bisection over the order-preserving keys of the values (counts over registers), the k chosen
// entries meet in LDS and each finds its place by counting.
#include "vocab_row.h"

namespace dcr {

namespace {

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }  // NaN -> -inf

}  // namespace

template <typename T, int NT, int EPT>
__global__ void __launch_bounds__(NT) topk_kernel(RowArgs r, int k, float inv_t,
                                                  float* __restrict__ values,
                                                  int* __restrict__ indices,
                                                  float* __restrict__ lse) {
  __shared__ float redf[NT / 64];
  __shared__ int redi[NT / 64];
  __shared__ float lv[kRowMaxK];
  __shared__ int li[kRowMaxK], count;
  const long n = blockIdx.x;
  const int tid = threadIdx.x, V = r.V;
  Row<T, NT, EPT> row(reinterpret_cast<const T*>(r.logits) + n * r.ld, V);

  float m = -INFINITY;
  int nan = 0;
  row.visit([&](int, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      nan |= x[j] != x[j];
      m = fmaxf(m, x[j]);
    }
  });
  m = block_reduce<NT>(m, redf, MaxOp());
  nan = block_reduce<NT>(nan, redi, AddOp());
  float sum = 0.f;
  row.visit([&](int, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += __expf((clean(x[j]) - m) * inv_t);
  });
  sum = block_reduce<NT>(sum, redf, AddOp());
  if (tid == 0) {
    lse[n] = nan ? __uint_as_float(0x7fc00000u)
                 : (m == INFINITY || m == -INFINITY) ? m : m * inv_t + __logf(sum);
    count = 0;
  }

  // count(>= lo) >= k > count(>= hi)
  unsigned lo = key_of(-INFINITY), hi = key_of(m) + 1;
  int above = 0, have = V;  // counts at hi and lo
  while (hi - lo > 1 && have != k) {
    const unsigned mid = lo + (hi - lo) / 2;
    const float f = float_of(mid);
    int c = 0;
    row.visit([&](int, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) c += x[j] >= f;
    });
    c = block_reduce<NT>(c, redi, AddOp());
    if (c >= k) lo = mid, have = c; else hi = mid, above = c;
  }
  const float cut = float_of(lo);
  int last = V - 1;  // entries equal to the cut are taken up to this column
  if (have != k) {   // more of them than places: the lowest columns
    const int need = k - above;
    int a = -1, b = V - 1;  // count(== cut, column <= b) >= need > count(.., column <= a)
    while (b - a > 1) {
      const int mid = a + (b - a) / 2;
      int c = 0;
      row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c += clean(x[j]) == cut && col + j <= mid;
      });
      c = block_reduce<NT>(c, redi, AddOp());
      if (c >= need) b = mid; else a = mid;
    }
    last = b;
  }
  __syncthreads();
  row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float y = clean(x[j]);
      if (y > cut || (y == cut && col + j <= last)) {
        const int at = atomicAdd(&count, 1);
        if (at < kRowMaxK) lv[at] = y, li[at] = col + j;
      }
    }
  });
  __syncthreads();
  for (int i = tid; i < k; i += NT) {
    const float y = lv[i];
    const int c = li[i];
    int at = 0;
    for (int j = 0; j < k; ++j) at += lv[j] > y || (lv[j] == y && li[j] < c);
    values[n * k + at] = y;
    indices[n * k + at] = c;
  }
}

void launch_topk(const RowArgs& r, int k, float inv_t, float* values, int* indices, float* lse,
                 hipStream_t s) {
#define CALL(NTH, E)                                                                         \
  if (r.is_bf16)                                                                             \
    topk_kernel<bf16, NTH, E><<<r.N, NTH, 0, s>>>(r, k, inv_t, values, indices, lse);        \
  else                                                                                       \
    topk_kernel<float, NTH, E><<<r.N, NTH, 0, s>>>(r, k, inv_t, values, indices, lse)
  DCR_ROW_DISPATCH(r.V, CALL);
#undef CALL
}

}  // namespace dcr
