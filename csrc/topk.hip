// The k largest logits of each row with their indices, and the row's log-sum-exp at a
// temperature: what a teacher records for distillation.  Order: value descending, ties by the
// lowest index; NaN counts as -inf in the order and makes the log-sum-exp NaN.
//
// One workgroup a row; the row is read once into registers, and that read is the bound.  From the
// maxima of groups of columns comes a value that at least k of the row reach; the some k entries
// that do meet in LDS, and each finds its place by counting those in front of it.  Rows of one wave
// with k over a quarter of their groups, and rows of many equal values, find the k-th largest
// value itself by halving a range of values, with counts by ballot.
//
// 32768 x 8192 fp32, k = 64: 241 us, 4.5 TB/s (a large copy reaches 5.0), the vector units busy for 82 %
// of it; k = 200 359 us, where the places of some 220 entries are the work.  10222 x 864 bf16, k = 31:
// 21 us of 4 for the read: one wave's chain of reductions a row; with k = 131, past a quarter of the
// groups, 77.
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
  constexpr bool kSmall = NT == 64;
  constexpr int kWaveGroups = EPT >= 16 ? 256 : 0;  // of a row of one wave
  __shared__ float redf[NT / 64];
  __shared__ int redi[NT / 64];
  constexpr int kCap = kSmall ? kRowMaxK : kList;
  __shared__ alignas(16) Entry list[kCap];
  __shared__ int count;
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
  if (!kSmall || 4 * k <= kWaveGroups) {
    const float f = reached_by<NT, kSmall ? (kWaveGroups ? kWaveGroups : 64) : kGroups>(
        row, gm, &reached, k);
    if (f > -INFINITY) {
      collect<NT>(row, list, &count, kCap, [&](float x, int) { return x >= f; });
      c = uniform(count);
    }
  }
  if (c < k || c > kCap) {
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
    if (tid == 0) count = 0;
    const Cut cut = cut_by_count<NT>(again, redi, m, low, k);
    __syncthreads();
    collect<NT>(again, list, &count, k, [&](float x, int col) {
      return x > cut.value || (x == cut.value && col <= cut.last);
    });
    c = k;
  }
  for (int i = tid; i < c; i += NT) {
    const Entry mine = list[i];
    const int at = place_of(list, c, mine);
    if (at < k) {
      values[n * k + at] = value_of(mine);
      indices[n * k + at] = column_of(mine);
    }
  }
}

// One wave takes a row of up to 1024 columns; longer rows get more threads before more registers,
// and past 65536 columns are read again instead of held.  Launches of a replayed graph over three sets of
// rows, us: 1024 x 65536, k = 64: bf16 71 held, 85 read again; fp32 123 held, although 88 of its registers
// go to scratch, 154 read again (the read alone takes 27 and 54).  2047 x 32001, k = 32, with 512 threads
// of 64 columns against 1024 of 32: bf16 50, 61; fp32 100, 94.  5296 x 12157, k = 9, with 512 threads of
// 32 columns against 256 of 64: bf16 61, 54; fp32 65, 71; 100 rows of it, fp32 8.7, 10.1.
template <typename T>
static void launch_type(const RowArgs& r, int k, float inv_t, float* values, int* indices,
                        float* lse, hipStream_t s) {
#define CALL(NTH, E) topk_kernel<T, NTH, E><<<r.N, NTH, 0, s>>>(r, k, inv_t, values, indices, lse)
  if (r.V <= 256) CALL(64, 4);
  else if (r.V <= 1024) CALL(64, 16);
  else if (r.V <= 4096) CALL(256, 16);
  else if (r.V <= 8192) CALL(256, 32);
  else if (r.V <= 16384) CALL(512, 32);
  else if (r.V <= 32768) CALL(512, 64);
  else if (r.V <= 65536) CALL(1024, 64);
  else CALL(1024, 0);
#undef CALL
}

void launch_topk(const RowArgs& r, int k, float inv_t, float* values, int* indices, float* lse,
                 hipStream_t s) {
  if (r.is_bf16) launch_type<bf16>(r, k, inv_t, values, indices, lse, s);
  else launch_type<float>(r, k, inv_t, values, indices, lse, s);
}

}  // namespace dcr
