// Sampling from filtered logits: one id a row from one uniform number a row.
//
// The row's tokens are ordered by value, ties by the lowest index, and weigh
// w_v = exp((l_v - max) / temperature).  Kept are the first top_k of the order; of these the
// tokens in front of which less than top_p of their weight lies; of these the ones with
// w >= min_p (the first of the order always).  Drawn is the first kept token, by index, at which
// the running weight passes u times the whole.  A temperature of 0 takes the first of the order.
// NaN counts as -inf; a row with nothing but -inf gives index 0.
//
// The answer is a whole number that a value next to a border decides, so weights are computed in
// 64 bits and added as whole numbers of 2^-44: sums are exact in any order, and a border is off
// by some 2^-44 of the largest weight a token.  2^44 times 262144 tokens fits 63 bits.
#include "vocab_row.h"

namespace dcr {

namespace {

typedef unsigned long long u64;
constexpr double kOne = 17592186044416.0;  // 2^44

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }
__device__ __forceinline__ float of_row(const PerRow& p, long n) { return p.p ? p.p[n] : p.v; }

struct Weigh {
  float m;
  double inv_t;
  __device__ __forceinline__ double real(float x) const {
    if (x == m) return 1.0;
    return x == -INFINITY || m == INFINITY ? 0.0 : exp(((double)x - (double)m) * inv_t);
  }
  __device__ __forceinline__ u64 operator()(float x) const { return (u64)(real(x) * kOne + 0.5); }
};

}  // namespace

template <typename T, int NT, int EPT>
__global__ void __launch_bounds__(NT) filter_sample_kernel(FilterArgs a) {
  constexpr int NW = NT / 64;
  constexpr int kMaxChunks = EPT ? EPT / 4 : kRowMaxV / (NT * 4);
  __shared__ float redf[NW];
  __shared__ int redi[NW];
  __shared__ u64 redu[NW];
  __shared__ u64 part[kMaxChunks * NW];
  __shared__ int found;
  __shared__ u64 left;
  const long n = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.r.V;
  Row<T, NT, EPT> row(reinterpret_cast<const T*>(a.r.logits) + n * a.r.ld, V);

  float m = -INFINITY;
  row.visit([&](int, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, x[j]);
  });
  m = block_reduce<NT>(m, redf, MaxOp());
  const float temp = of_row(a.temperature, n);
  if (!(temp > 0.f) || m == -INFINITY) {  // the first of the order
    int at = V;
    row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (clean(x[j]) == m) at = min(at, col + j);
    });
    at = block_reduce<NT>(at, redi, MinOp());
    if (tid == 0) a.out[n] = at;
    return;
  }
  const Weigh weigh{m, 1.0 / (double)temp};
  const float top_p = of_row(a.top_p, n), min_p = of_row(a.min_p, n);
  const int want = a.top_k ? a.top_k[n] : a.top_k_all;

  // kept so far: values above `cut`, and those equal to it up to column `last`
  float cut = -INFINITY;
  int last = V - 1;
  auto kept = [&](float x, int col) { return x > cut || (x == cut && col <= last); };
  // the column of the need-th kept value equal to f
  auto nth_equal = [&](float f, long need) {
    int lo = -1, hi = last;
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      int c = 0;
      row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c += clean(x[j]) == f && col + j <= mid;
      });
      c = block_reduce<NT>(c, redi, AddOp());
      if (c >= need) hi = mid; else lo = mid;
    }
    return hi;
  };

  if (want > 0 && want < V) {
    unsigned lo = key_of(-INFINITY), hi = key_of(m) + 1;
    int above = 0, have = V;
    while (hi - lo > 1 && have != want) {
      const unsigned mid = lo + (hi - lo) / 2;
      const float f = float_of(mid);
      int c = 0;
      row.visit([&](int, float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c += x[j] >= f;
      });
      c = block_reduce<NT>(c, redi, AddOp());
      if (c >= want) lo = mid, have = c; else hi = mid, above = c;
    }
    const float f = float_of(lo);
    if (have != want) last = nth_equal(f, want - above);
    cut = f;
  }
  auto mass = [&](auto&& pred) {
    u64 s = 0;
    row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = clean(x[j]);
        if (kept(y, col + j) && pred(y)) s += weigh(y);
      }
    });
    return block_reduce<NT>(s, redu, AddOp());
  };
  if (top_p < 1.0f) {
    const double target = (double)top_p * (double)mass([](float) { return true; });
    // mass(>= lo) >= target > mass(>= hi)
    unsigned lo = max(key_of(cut), key_of(-INFINITY)), hi = key_of(m) + 1;
    u64 above = 0;
    while (hi - lo > 1) {
      const unsigned mid = lo + (hi - lo) / 2;
      const float f = float_of(mid);
      const u64 s = mass([&](float x) { return x >= f; });
      if ((double)s >= target) lo = mid; else hi = mid, above = s;
    }
    const float f = float_of(lo);
    // of the values equal to f, those in front of which less than the target lies
    const double need = ceil((target - (double)above) / (double)weigh(f));
    const int most = f == cut ? last : V - 1;
    int equal = 0;
    row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) equal += clean(x[j]) == f && col + j <= most;
    });
    equal = block_reduce<NT>(equal, redi, AddOp());
    last = most;
    if (need < (double)equal) last = nth_equal(f, need < 1.0 ? 1 : (long)need);
    cut = f;
  }

  // ---- the draw: sums of a wave's chunk, in the order of the columns
  const double floor_w = min_p > 1.0f ? 1.0 : (double)min_p;  // (NaN: no floor)
  auto weight = [&](float x, int col) -> u64 {
    if (!kept(x, col)) return 0;
    const double q = weigh.real(x);
    return q < floor_w ? 0 : (u64)(q * kOne + 0.5);
  };
  u64 total = 0;
  row.visit([&](int col, float (&x)[4], int c) {
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) s += weight(clean(x[j]), col + j);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) part[c * NW + w] = s;
    total += s;
  });
  if (lane != 0) total = 0;
  total = block_reduce<NT>(total, redu, AddOp());
  __syncthreads();
  double u = (double)a.u[n];
  if (!(u > 0.0)) u = 0.0;
  const double at = u * (double)total;
  u64 r = at < (double)total ? (u64)at : total - 1;
  if (r >= total) r = total - 1;
  if (w == 0) {  // the wave and chunk that holds it
    const int np = row.chunks() * NW, per = (np + 63) / 64;
    u64 s = 0;
    for (int i = lane * per; i < min((lane + 1) * per, np); ++i) s += part[i];
    u64 upto = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    u64 before = upto - s;
    if (r >= before && r < upto) {
      int i = lane * per;
      while (r >= before + part[i]) before += part[i++];
      found = i;
      left = r - before;
    }
  }
  __syncthreads();
  const int fc = found / NW, fw = found % NW;
  const u64 rr = left;
  if (w == fw)
    row.visit([&](int col, float (&x)[4], int c) {
      if (c != fc) return;
      u64 q[4], s = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += q[j] = weight(clean(x[j]), col + j);
      u64 upto = s;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(upto, o, 64);
        if (lane >= o) upto += y;
      }
      u64 before = upto - s;
      if (rr >= before && rr < upto) {
        int pick = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (rr >= before && rr < before + q[j]) pick = col + j;
          before += q[j];
        }
        a.out[n] = pick;
      }
    });
}

void launch_filter_sample(const FilterArgs& a, hipStream_t s) {
#define CALL(NTH, E)                                                         \
  if (a.r.is_bf16) filter_sample_kernel<bf16, NTH, E><<<a.r.N, NTH, 0, s>>>(a); \
  else filter_sample_kernel<float, NTH, E><<<a.r.N, NTH, 0, s>>>(a)
  DCR_ROW_DISPATCH(a.r.V, CALL);
#undef CALL
}

}  // namespace dcr
