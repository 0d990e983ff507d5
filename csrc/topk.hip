// The k largest logits of each row with their indices, and the row's log-sum-exp at a
// temperature: what a teacher records for distillation.  Order: value descending, ties by the
// lowest index; NaN counts as -inf in the order and makes the log-sum-exp NaN.
//
// One workgroup a row; the row is read once into registers, and that read is the bound.  Up to
// 1024 columns (one wave) the k-th largest value is found by halving a range of values, with
// counts by ballot.  Larger rows first find a value that at least k of them reach, from the maxima
// of 1024 groups of columns; the some k entries that reach it meet in LDS.  Each collected entry
// finds its place by counting those in front of it.
#include "vocab_row.h"

namespace dcr {

namespace {

constexpr int kList = 1024;  // entries that meet in LDS; more (many equal values) are cut first

}  // namespace

template <typename T, int NT, int EPT>
__global__ void __launch_bounds__(NT) topk_kernel(RowArgs r, int k, float inv_t,
                                                  float* __restrict__ values,
                                                  int* __restrict__ indices,
                                                  float* __restrict__ lse) {
  constexpr bool kSmall = NT == 64 && EPT <= 16;
  __shared__ float redf[NT / 64];
  __shared__ int redi[NT / 64];
  constexpr int kCap = kSmall ? kRowMaxK : kList;
  __shared__ float lv[kCap];
  __shared__ int li[kCap], count;
  __shared__ float gm[NT == 64 ? 1 : kGroups], reached;
  const long n = blockIdx.x;
  const int tid = threadIdx.x, V = r.V;
  const float log2e_t = inv_t * 1.44269504088896341f;
  const T* z = reinterpret_cast<const T*>(r.logits) + n * r.ld;
  Row<T, NT, EPT> row(z, V);

  float m = -INFINITY;
  row.visit([&](int, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, x[j]);
  });
  if (tid == 0) count = 0;
  m = block_reduce<NT>(m, redf, MaxOp());
  if (m > -INFINITY && m < INFINITY) {
    float sum = 0.f;
    row.visit([&](int, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += __builtin_amdgcn_exp2f((x[j] - m) * log2e_t);
    });
    sum = block_reduce<NT>(sum, redf, AddOp());  // (NaN where the row holds one)
    if (tid == 0) lse[n] = m * inv_t + __logf(sum);
  } else {
    int nan = 0;
    row.visit([&](int, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) nan |= x[j] != x[j];
    });
    nan = __syncthreads_or(nan);
    if (tid == 0) lse[n] = nan ? __uint_as_float(0x7fc00000u) : m;
  }

  int c = 0;  // collected entries
  if constexpr (!kSmall) {
    const float f = reached_by<NT>(row, gm, &reached, k);
    if (f > -INFINITY) {
      collect<NT>(row, lv, li, &count, kList, [&](float x, int) { return x >= f; });
      c = uniform(count);
    }
  }
  if (c < k || c > kList) {
    // hardly ever for the long rows: they are read again rather than hold registers for it
    auto again = [&] {
      if constexpr (kSmall) return row;
      else return Row<T, NT, 0>(z, V);
    }();
    float low = INFINITY;
    again.visit([&](int, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > -INFINITY) low = fminf(low, x[j]);
    });
    low = block_reduce<NT>(low, redf, MinOp());
    if (!kSmall && tid == 0) count = 0;
    const Cut cut = cut_by_count<NT>(again, redi, m, low, k);
    __syncthreads();
    collect<NT>(again, lv, li, &count, k, [&](float x, int col) {
      return x > cut.value || (x == cut.value && col <= cut.last);
    });
    c = k;
  }
  for (int i = tid; i < c; i += NT) {
    const float y = lv[i];
    const int col = li[i];
    int at = 0;
#pragma unroll 8
    for (int j = 0; j < c; ++j) at += lv[j] > y || (lv[j] == y && li[j] < col);
    if (at < k) {
      values[n * k + at] = y;
      indices[n * k + at] = col;
    }
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
