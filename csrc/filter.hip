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
//
// One workgroup a row, the row in registers: it is read once.  Three ways to the kept set:
//   top_k <= 256      the first top_k meet in LDS and are ordered there (as in topk.hip); only
//                     they are weighed.
//   top_p, large top_k  counts and weights by value interval (kBins of them, in LDS) find the
//                     interval that holds a border; its entries meet in LDS, are ordered, and the
//                     border is the one entry in front of which less than the target lies.
//   otherwise         nothing to find: min_p is a bound on the value.
// 256 rows of 32001 bf16: all kept 21 us, top_k 50 17, top_p 42, every row with settings of its own 47
// (the read alone is 3 us): one workgroup a CU, its vector units busy for a third of that; weighing every
// token in 64 bits, once or twice, and for top_p an LDS addition each, take their turns with barriers and
// scans.  One row takes nearly as long: 17, 14, 38.  16 rows of 65: 7.3 us a call, nearly all of it the
// one wave's chain of selection and scans.
//
// An interval that holds more than kList entries is halved by values until one value is left, as a
// whole, some 30 visits of the row: rows of many equal values, and flat rows with a finite mask.  The
// intervals cover what lies within 32 T of the largest value or, if that is less, everything above
// -inf, and a mask of the lowest finite value is part of that.  64 x 32001 fp32 of deviation 0.25, every
// third token masked, top_p 0.9: 41 us masked with -inf, 69 with the lowest value; 64 x 131072 of
// deviation 1: 142 and 2000.
#include "vocab_row.h"

namespace dcr {

namespace {

typedef unsigned long long u64;
constexpr int kList = 1024;

__device__ __forceinline__ float of_row(const PerRow& p, long n) { return p.p ? p.p[n] : p.v; }

// 2^44 exp((x - m) / temperature), as a number and rounded.  2^f on [-1/2, 1/2] by its power
// series to f^11 (the rest is below 2^-47); adding 2^52 leaves the rounded number in the low bits.
// No branches: -inf (and the NaN of its product with a c of 0) ends at 2^-64, which rounds to 0, and a
// row with +inf counts from 1e300, where all else ends there too.
struct Weigh {
  double top, c;  // c = log2(e) / temperature
  __device__ __forceinline__ Weigh(float m, float temp)
      : top(m == INFINITY ? 1e300 : (double)m), c(fmax(1.4426950408889634 / (double)temp, 1e-280)) {}
  __device__ __forceinline__ double real(float x) const {
    const double y = fmin(fmax(((double)x - top) * c, -64.0), 0.0);
    const double n = rint(y), f = y - n;
    double p = 4.4455382718708114e-10;  // ln(2)^k / k!, k = 11 .. 0
    p = fma(p, f, 7.0549116208011234e-09);
    p = fma(p, f, 1.0178086009239699e-07);
    p = fma(p, f, 1.3215486790144307e-06);
    p = fma(p, f, 1.5252733804059841e-05);
    p = fma(p, f, 1.5403530393381608e-04);
    p = fma(p, f, 1.3333558146428443e-03);
    p = fma(p, f, 9.6181291076284772e-03);
    p = fma(p, f, 5.5504108664821580e-02);
    p = fma(p, f, 2.4022650695910071e-01);
    p = fma(p, f, 6.9314718055994531e-01);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n + 44);
  }
  __device__ __forceinline__ u64 whole(double w) const {
    return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 operator()(float x) const { return whole(real(x)); }
};

// The threads of a workgroup take `c` entries together, kTeam threads each; f(entry, member)
// returns a member's share of a sum, g(entry, sum) runs in every member.
template <int NT, typename T, typename F, typename G>
__device__ __forceinline__ void by_teams(int c, F&& f, G&& g) {
  constexpr int kTeam = NT == 64 ? 1 : NT == 256 ? 2 : 4;
  for (int i = threadIdx.x / kTeam; i - (int)threadIdx.x / kTeam < c; i += NT / kTeam) {
    T x = i < c ? f(i, (int)threadIdx.x % kTeam, kTeam) : T(0);
    if (kTeam > 1) x += dpp<0xB1>(x);
    if (kTeam > 2) x += dpp<0x4E>(x);
    if (i < c) g(i, x);
  }
}

struct alignas(16) Weighed { Entry e; u64 w; };

template <int NT>
struct Work {  // LDS of one workgroup
  static constexpr int kBins = NT == 64 ? 256 : 1024;
  static constexpr int kCap = NT == 64 ? 256 : kList;
  float redf[NT / 64];
  int redi[NT / 64];
  u64 redu[NT / 64];
  alignas(16) Entry list[kCap];
  u64 lw[kCap];
  union {
    struct { u64 mass[kBins]; int count[kBins]; } bin;
    Weighed top[kRowMaxK];  // ordered entries
    float gm[NT == 64 ? 1 : kGroups];
  };
  int n, chosen, chosen_last;
  float reached, chosen_value;
  u64 chosen_mass, chosen_total;
  int bin_at, bin_count;
  u64 bin_mass;
};

// The bin in which the running number (of entries, or of weight) from bin 0 on reaches `target`:
// s.bin_at, and what lies in front of it in s.bin_count / s.bin_mass.  s.bin_at is kBins if it is
// never reached.
template <int NT, bool BY_MASS>
__device__ __forceinline__ void find_bin(Work<NT>& s, u64 target) {
  constexpr int kPer = Work<NT>::kBins / 64;
  if (threadIdx.x == 0) s.bin_at = Work<NT>::kBins;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int b0 = threadIdx.x * kPer;
    int c = 0;
    u64 w = 0;
    for (int i = 0; i < kPer; ++i) c += s.bin.count[b0 + i], w += s.bin.mass[b0 + i];
    int cb = wave_scan(c) - c;
    u64 wb = wave_scan(w) - w;
    const u64 from = BY_MASS ? wb : (u64)cb, to = from + (BY_MASS ? w : (u64)c);
    if (from < target && target <= to) {
      int i = b0;
      for (; i < b0 + kPer - 1; ++i) {
        const u64 next = BY_MASS ? wb + s.bin.mass[i] : (u64)(cb + s.bin.count[i]);
        if (next >= target) break;
        cb += s.bin.count[i];
        wb += s.bin.mass[i];
      }
      s.bin_at = i;
      s.bin_count = cb;
      s.bin_mass = wb;
    }
  }
  __syncthreads();
}

// chunks of four a thread that a row in LDS may take: 32 KB for 256 threads, 128 KB for 1024
template <typename T, int NT>
constexpr int lds_chunks() { return (NT == 256 ? 32768 : 131072) / (NT * 4 * (int)sizeof(T)); }

}  // namespace

// EPT: elements a thread in registers; 0: the row is read again by every visit; -1: it is in LDS
template <typename T, int NT, int EPT>
__global__ void __launch_bounds__(NT) filter_sample_kernel(FilterArgs a) {
  constexpr int NW = NT / 64, kBins = Work<NT>::kBins, kCap = Work<NT>::kCap;
  constexpr int kMaxChunks = EPT > 0 ? EPT / 4 : EPT < 0 ? lds_chunks<T, NT>() : kRowMaxV / (NT * 4);
  extern __shared__ char held[];
  __shared__ Work<NT> s;
  __shared__ u64 part[kMaxChunks * NW];
  const long n = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.r.V;
  const T* logits = reinterpret_cast<const T*>(a.r.logits) + n * a.r.ld;
  auto row = [&] {
    if constexpr (EPT < 0) return RowLds<T, NT>(logits, V, held);
    else return Row<T, NT, EPT>(logits, V);
  }();

  float m = -INFINITY, low = INFINITY;
  row.visit([&](int, float (&x)[4], int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m = fmaxf(m, x[j]);
      if (x[j] > -INFINITY) low = fminf(low, x[j]);
    }
  });
  if (tid == 0) s.n = 0;
  m = block_reduce<NT>(m, s.redf, MaxOp());
  const float temp = uniform(of_row(a.temperature, n));
  if (!(temp > 0.f) || m == -INFINITY) {  // the first of the order
    int at = V;
    row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (clean(x[j]) == m) at = min(at, col + j);
    });
    at = block_reduce<NT>(at, s.redi, MinOp());
    if (tid == 0) a.out[n] = at;
    return;
  }
  low = block_reduce<NT>(low, s.redf, MinOp());
  const Weigh weigh(m, temp);
  const float top_p = uniform(of_row(a.top_p, n)), min_p = of_row(a.min_p, n);
  const int want = uniform(a.top_k ? a.top_k[n] : a.top_k_all);
  // (a NaN min_p: no floor)
  const double floor_w = (min_p > 1.0f ? 1.0 : (double)min_p) * 17592186044416.0;
  double u = (double)a.u[n];
  if (!(u > 0.0)) u = 0.0;
  auto place = [&](u64 total) {  // u of the whole; total is at least the first's 2^44
    const double at = u * (double)total;
    const u64 r = at < (double)total ? (u64)at : total - 1;
    return r < total ? r : total - 1;
  };
  // the least whole number that is not below p of the total (at least 1: the first is kept)
  auto share = [&](u64 total) {
    const double t = ceil((double)top_p * (double)total);
    return t >= 1.0 ? (u64)t : (u64)1;
  };

  if (want > 0 && want <= kRowMaxK && want < V) {
    // ---- the first `want`, ordered in LDS
    int c = kCap + 1;
    constexpr int kWaveGroups = EPT >= 16 ? 256 : 0;  // of a row of one wave
    if (NT != 64 || 4 * want <= kWaveGroups) {
      const float f = reached_by<NT, NT == 64 ? (kWaveGroups ? kWaveGroups : 64) : kGroups>(
          row, s.gm, &s.reached, want);
      // (entries of -inf weigh nothing: fewer than `want` others are all that is needed)
      collect<NT>(row, s.list, &s.n, kCap, [&](float x, int) {
        return x >= f && x > -INFINITY;
      });
      c = uniform(s.n);
    }
    if (c > kCap) {
      const Cut cut = cut_by_count<NT>(row, s.redi, m, low, want);
      if (tid == 0) s.n = 0;
      __syncthreads();
      collect<NT>(row, s.list, &s.n, kCap, [&](float x, int col) {
        return x > -INFINITY && (x > cut.value || (x == cut.value && col <= cut.last));
      });
      c = uniform(s.n);
    }
    by_teams<NT, int>(
        c,
        [&](int i, int k, int K) {
          const Entry mine = s.list[i];
          const int part = ((c + K - 1) / K + 1) & ~1, from = k * part;  // pairs stay together
          return place_of(s.list + from, max(0, min(c - from, part)), mine);
        },
        [&](int i, int at) {
          if (at < want) {
            const Entry mine = s.list[i];
            s.top[at] = Weighed{mine, weigh(value_of(mine))};
          }
        });
    c = min(c, want);
    __syncthreads();
    if (w == 0) {
      constexpr int kPer = kRowMaxK / 64;
      u64 q[kPer], sum = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = lane * kPer + i;
        q[i] = at < c ? s.top[at].w : 0;
        sum += q[i];
      }
      u64 before = wave_scan(sum) - sum;
      const u64 total = lane_value(before + sum, 63);
      const u64 target = top_p < 1.0f ? share(total) : ~0ull;
      int kept = 0;
      u64 mass = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = lane * kPer + i;
        const bool in = at < c && before < target &&
                        (at == 0 || !(weigh.real(value_of(s.top[at].e)) < floor_w));
        before += q[i];
        if (in) kept = at + 1, mass += q[i];
      }
      kept = wave_reduce(kept, MaxOp());
      mass = wave_reduce(mass, AddOp());
      if (lane == 0) s.chosen = kept, s.chosen_total = mass;
    }
    __syncthreads();
    c = uniform(s.chosen);
    const u64 r = place(s.chosen_total);
    by_teams<NT, u64>(  // running weights in the order of the indices
        c,
        [&](int i, int k, int K) {
          const unsigned col = (unsigned)s.top[i].e;  // (its complement: larger for lower columns)
          u64 before = 0;
#pragma unroll 8
          for (int j = k; j < c; j += K) {
            const Weighed q = s.top[j];
            before += (unsigned)q.e > col ? q.w : 0;
          }
          return before;
        },
        [&](int i, u64 before) {
          if (r >= before && r < before + s.top[i].w) a.out[n] = column_of(s.top[i].e);
        });
    return;
  }

  // kept so far: values above `cut`, and those equal to it up to column `last`
  float cut = -INFINITY;
  int last = V - 1;
  auto kept = [&](float x, int col) { return x > cut || (x == cut && col <= last); };
  const bool by_k = want > 0 && want < V, by_p = top_p < 1.0f;
  if (by_k || by_p) {
    // ---- counts and weights of kBins intervals of x = (m - l) / temperature; from 32 on the
    // weight rounds to 0, so where the intervals end there, what the last one drops is never drawn
    const float inv_t = 1.0f / temp;
    const float span = fminf((m - low) * inv_t, 32.0f);
    const float per = span > 0.f ? (float)kBins / span : 0.f;
    const bool clipped = !((m - low) * inv_t < 32.0f);
    auto bin_of = [&](float x) {
      if (x == m) return 0;
      const float d = (m - x) * inv_t * per;  // falls with x, also as rounded
      return d < (float)(kBins - 1) ? (int)d : kBins - 1;
    };
    for (int i = tid; i < kBins; i += NT) s.bin.count[i] = 0, s.bin.mass[i] = 0;
    __syncthreads();
    row.visit([&](int, float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > -INFINITY) {
          const int b = bin_of(x[j]);
          const u64 q = weigh(x[j]);
          if (by_k) atomicAdd(&s.bin.count[b], 1);
          if (q) atomicAdd(&s.bin.mass[b], q);
        }
    });
    __syncthreads();
    // the entry of a bin in front of which (with what lies in front of the bin) less than
    // `target` entries or weight lies, and with which it does not: the last one kept
    auto border = [&](int b, u64 in_front, u64 target, bool by_mass) {
      if (tid == 0) s.n = 0;
      __syncthreads();
      collect<NT>(row, s.list, &s.n, kCap, [&](float x, int col) {
        return x > -INFINITY && bin_of(x) == b && kept(x, col);
      });
      const int c = uniform(s.n);
      if (c <= kCap) {
        for (int i = tid; i < c; i += NT) s.lw[i] = weigh(value_of(s.list[i]));
        __syncthreads();
        by_teams<NT, u64>(
            c,
            [&](int i, int k, int K) {
              const Entry mine = s.list[i];
              u64 front = 0;
#pragma unroll 8
              for (int j = k; j < c; j += K)
                front += s.list[j] > mine ? (by_mass ? s.lw[j] : 1) : 0;
              return front;
            },
            [&](int i, u64 front) {
              const u64 before = in_front + front;
              if (before < target && target <= before + (by_mass ? s.lw[i] : 1)) {
                s.chosen_value = value_of(s.list[i]);
                s.chosen_last = column_of(s.list[i]);
              }
            });
        __syncthreads();
        cut = uniform(s.chosen_value);
        last = uniform(s.chosen_last);
        u64 mass = 0;
        for (int i = tid; i < c; i += NT) {
          const float y = value_of(s.list[i]);
          if (kept(y, column_of(s.list[i]))) mass += s.lw[i];
        }
        return block_reduce<NT>(mass, s.redu, AddOp());
      }
      // many entries: halve the bin's range of values
      auto amount = [&](float f) {
        u64 q = 0;
        row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (x[j] >= f && x[j] > -INFINITY && bin_of(x[j]) == b &&
                kept(x[j], col + j))
              q += by_mass ? weigh(x[j]) : 1;
        });
        return block_reduce<NT>(q, s.redu, AddOp());
      };
      unsigned lo = key_of(low), hi = key_of(m) + 1;
      u64 above = 0;  // amount(>= hi) in front of the target, which amount(>= lo) reaches
      for (int round = 0; hi - lo > 1; ++round) {
        const unsigned mid = split_key(lo, hi, round);
        const u64 q = amount(float_of(mid));
        if (in_front + q >= target) lo = mid; else hi = mid, above = q;
      }
      const float f = float_of(lo);
      const u64 each = by_mass ? weigh(f) : 1;
      const u64 need = (target - in_front - above + each - 1) / each;  // entries equal to f
      int c0 = -1, c1 = V - 1;
      while (c1 - c0 > 1) {
        const int mid = c0 + (c1 - c0) / 2;
        const int q = count_if<NT>(row, s.redi, [&](float x, int col) {
          return x == f && col <= mid && kept(x, col);
        });
        if ((u64)q >= need) c1 = mid; else c0 = mid;
      }
      u64 mass = 0;
      row.visit([&](int col, float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (x[j] > -INFINITY && bin_of(x[j]) == b && kept(x[j], col + j) &&
              (x[j] > f || (x[j] == f && col + j <= c1)))
            mass += weigh(x[j]);
      });
      mass = block_reduce<NT>(mass, s.redu, AddOp());
      cut = f;
      last = c1;
      return mass;
    };
    u64 total = 0;  // the weight of the first top_k
    bool all = !by_k;
    if (by_k) {
      find_bin<NT, false>(s, (u64)want);
      const int b = uniform(s.bin_at);
      // (fewer than top_k above -inf, or the rest weighs nothing: all weight is kept)
      all = b == kBins || (clipped && b == kBins - 1);
      if (!all) {
        const u64 front = uniform(s.bin_mass);
        total = front + border(b, (u64)uniform(s.bin_count), (u64)want, false);
      }
    }
    if (by_p) {
      if (all) {
        u64 q = 0;
        for (int i = tid; i < kBins; i += NT) q += s.bin.mass[i];
        total = block_reduce<NT>(q, s.redu, AddOp());
      }
      const u64 target = share(total);
      find_bin<NT, true>(s, target);
      const int b = uniform(s.bin_at);
      if (b < kBins) border(b, uniform(s.bin_mass), target, true);
    }
  }

  // ---- the draw, in the order of the columns: the weight of each wave's chunks, then the lane
  const bool cut_off = cut > -INFINITY || last < V - 1, floored = floor_w > 0.0;
  auto weights = [&](const float (&x)[4], int col, u64 (&q)[4]) {
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      in[j] = !cut_off || kept(clean(x[j]), col + j);
      q[j] = 0;
    }
    if (!__any(in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double f = weigh.real(clean(x[j]));
      q[j] = in[j] && !(floored && f < floor_w) ? weigh.whole(f) : 0;
    }
  };
  u64 total = 0;
  row.visit([&](int col, float (&x)[4], int c) {
    u64 four[4];
    weights(x, col, four);
    u64 q = four[0] + four[1] + four[2] + four[3];
    if (__any(q != 0)) q = wave_reduce(q, AddOp());
    total += q;
    if (lane == 0) part[c * NW + w] = q;
  });
  if (lane != 0) total = 0;
  total = block_reduce<NT>(total, s.redu, AddOp());
  __syncthreads();
  const u64 r = place(total);
  if (w == 0) {  // the wave and chunk that holds it
    const int np = row.chunks() * NW, per = (np + 63) / 64;
    u64 q = 0;
    for (int i = lane * per; i < min((lane + 1) * per, np); ++i) q += part[i];
    u64 before = wave_scan(q) - q;
    if (r >= before && r < before + q) {
      int i = lane * per;
      while (r >= before + part[i]) before += part[i++];
      s.chosen = i;
      s.chosen_mass = r - before;
    }
  }
  __syncthreads();
  const int at = uniform(s.chosen), fc = at / NW, fw = at % NW;
  const u64 rest = uniform(s.chosen_mass);
  if (w == fw)
    row.visit([&](int col, float (&x)[4], int c) {
      if (c != fc) return;
      u64 q[4];
      weights(x, col, q);
      const u64 sum = q[0] + q[1] + q[2] + q[3];
      u64 before = wave_scan(sum) - sum;
      if (rest >= before && rest < before + sum) {
        int pick = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (rest >= before && rest < before + q[j]) pick = col + j;
          before += q[j];
        }
        a.out[n] = pick;
      }
    });
}

template <typename T>
static void launch_type(const FilterArgs& a, hipStream_t s) {
  const int V = a.r.V;
  auto lds = [&](int nt) { return (size_t)((V + nt * 4 - 1) / (nt * 4)) * nt * 4 * sizeof(T); };
#define CALL(NTH, E, LDS) filter_sample_kernel<T, NTH, E><<<a.r.N, NTH, LDS, s>>>(a)
  if (V <= 256) CALL(64, 4, 0);
  else if (V <= 1024) CALL(64, 16, 0);
  else if (lds(256) <= 32768) CALL(256, -1, lds(256));
  else if (lds(1024) <= 131072) {
    if (lds(1024) > 32768)
      hipFuncSetAttribute(reinterpret_cast<const void*>(&filter_sample_kernel<T, 1024, -1>),
                          hipFuncAttributeMaxDynamicSharedMemorySize, 131072);
    CALL(1024, -1, lds(1024));
  }
  else CALL(1024, 0, 0);
#undef CALL
}

void launch_filter_sample(const FilterArgs& a, hipStream_t s) {
  if (a.r.is_bf16) launch_type<bf16>(a, s); else launch_type<float>(a, s);
}

}  // namespace dcr
