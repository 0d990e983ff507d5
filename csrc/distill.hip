// Distillation from a teacher's recorded top logits: loss and gradient in one pass over the
// student's logits, beside the cross-entropy of xent.hip.
//
// With the student's p = softmax(z / T) and the teacher's recorded entries (i_j, t_j):
//   q_j = exp(t_j / T - lse), r = max(0, 1 - sum q_j)   with the teacher's log-sum-exp at T, or
//   q   = softmax_j(t_j / T), r = 0                     without it
//   no divergence, where all t_j are -inf and the log-sum-exp is, or is not given
//   loss = alpha T^2 [sum_j q_j (log q_j - log p_{i_j}) + r (log r - log s)]
//        + (1 - alpha) (lse(z) - z_y),                  s = the student's mass off the entries
//   d/dz_v = alpha T (p_v - q_v)            at the entries
//            alpha T p_v (1 - r / s)        elsewhere
//            + (1 - alpha) (softmax(z)_v - [v = y])
//
// One workgroup a row, the row in registers, so z is read once and the gradient written once:
// that traffic is the bound of long fp32 rows, the issue of vector instructions of bf16 ones.  The recorded columns are marked in an LDS bitmap; their threads
// hold them apart (they write those gradients too), and the rest has a maximum and sum of its
// own.  So s is never a difference 1 - sum p, which has no digits left where the student is sure.
//
// A divergence is a small sum of large terms of both signs.  With sum q + r = sum p + s = 1 it is
// also the sum of q (d - 1 + exp(-d)), d = log(q / p), over the entries and the rest: no term is
// negative, none cancels another, and a common error of the log-probabilities drops out.  For the
// same reason 1 - r / s is taken as sum (q - p) / s where the entries hold little.
#include "vocab_row.h"

namespace dcr {

namespace {

// d - 1 + exp(-d) = d^2/2! - d^3/3! + ..., up to |d| = 1 (the rest is below 2^-31 of it)
__device__ __forceinline__ float excess(float d) {
  float p = 2.0876756987868099e-9f;  // 1 / 12!
  p = __builtin_fmaf(p, -d, 2.5052108385441719e-8f);
  p = __builtin_fmaf(p, -d, 2.7557319223985891e-7f);
  p = __builtin_fmaf(p, -d, 2.7557319223985891e-6f);
  p = __builtin_fmaf(p, -d, 2.4801587301587302e-5f);
  p = __builtin_fmaf(p, -d, 1.9841269841269841e-4f);
  p = __builtin_fmaf(p, -d, 1.3888888888888889e-3f);
  p = __builtin_fmaf(p, -d, 8.3333333333333333e-3f);
  p = __builtin_fmaf(p, -d, 4.1666666666666667e-2f);
  p = __builtin_fmaf(p, -d, 1.6666666666666667e-1f);
  p = __builtin_fmaf(p, -d, 0.5f);
  return p * d * d;
}
// q d - q + p, for q > 0
__device__ __forceinline__ float term(float q, float p, float d) {
  return fabsf(d) <= 1.0f ? q * excess(d) : q * (d - 1.0f) + p;
}

}  // namespace

template <typename T, typename G, int NT, int EPT>
__global__ void __launch_bounds__(NT) distill_kernel(DistillArgs a) {
  constexpr int kE = NT < kRowMaxK ? kRowMaxK / NT : 1;  // entries a thread
  extern __shared__ unsigned bits[];
  __shared__ float red[(3 + 5 + 3) * (NT / 64)];
  __shared__ int ei[kRowMaxK], twice;
  __shared__ float eq[kRowMaxK];  // q of the entries, for columns recorded twice
  const long n = blockIdx.x;
  const int tid = threadIdx.x, V = a.r.V, k = a.k;
  const T* z = reinterpret_cast<const T*>(a.r.logits) + n * a.r.ld;
  G* grad = a.grad ? reinterpret_cast<G*>(a.grad) + n * a.grad_ld : nullptr;
  const float inv_t = a.inv_t, c_t = a.log2e_t;
  constexpr float c_1 = 1.44269504088896341f;
  const int y = a.targets ? a.targets[n] : -1;
  const bool skip = a.targets && (y < 0 || y >= V);
  const bool ce = a.targets && a.alpha < 1.0f;
  const bool two = ce && inv_t != 1.0f;
  // x / T - y with one rounding: 1 / T is a sum of two numbers.  (For the entries, whose terms are told
  // apart by d = log(q / p); the columns off them take one rounded log2(e) / T and the exponential of
  // the hardware: a few units of 2^-24 and |z - max| / T of them.)
  auto scaled = [&](float x, float y) {
    return x == -INFINITY ? x : __builtin_fmaf(x, inv_t, __builtin_fmaf(x, a.inv_t_low, -y));
  };
  // a second exponential an element

  // ---- the entries: column (-1: none), t, the student's z
  int i_e[kE];
  float t_e[kE], z_e[kE];
  bool first[kE];  // the first entry of its column
  // (k is uniform: a wave passes over the entries that none of it has)
#define DCR_ENTRIES(e) for (int e = 0; e < kE && (e == 0 || e * NT < k); ++e)
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    const int j = e * NT + tid;
    i_e[e] = j < k ? a.indices[n * k + j] : -1;
    if (i_e[e] >= V) i_e[e] = -1;
    t_e[e] = i_e[e] >= 0 ? a.values[n * k + j] : -INFINITY;
    z_e[e] = -INFINITY;
    first[e] = false;
  }
  const float z_y = ce && !skip ? (float)z[y] : 0.f;
  Row<T, NT, EPT> row(z, V);
  for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
  if (tid == 0) twice = 0;
  __syncthreads();
#pragma unroll
  DCR_ENTRIES(e) {
    const int i = i_e[e];
    first[e] = i >= 0;
    z_e[e] = i >= 0 ? (float)z[i] : -INFINITY;
    if (i >= 0 && (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31) & 1)) twice = 1;
    if (e * NT + tid < k) ei[e * NT + tid] = i;
  }
  __syncthreads();
  if (twice) {  // a column recorded more than once: its first entry stands for it
#pragma unroll
    for (int e = 0; e < kE; ++e)
      for (int j = 0; j < e * NT + tid && first[e]; ++j)
        if (ei[j] == i_e[e]) first[e] = false;
  }
  // the entries' nibble of four columns
  auto marked = [&](int col) -> unsigned {
    return col < V ? bits[col >> 5] >> (col & 31) & 15u : 0u;
  };
  auto rest_of = [&](float (&x)[4], int col) {  // a row that is read again loses them each time
    if constexpr (EPT == 0) {
      const unsigned q = marked(col);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (q >> j & 1) x[j] = -INFINITY;
    }
  };
  if constexpr (EPT > 0) row.erase(marked);

  // ---- maxima: of the rest, of the entries' z and t
  float top[3] = {-INFINITY, -INFINITY, -INFINITY};
  // sums at T and at 1: of the rest, of the entries' z; and of the entries' t
  float sum[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float (&x)[4], float over) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum[0] += __builtin_amdgcn_exp2f((x[j] - over) * c_t);
      if (two) sum[1] += __builtin_amdgcn_exp2f((x[j] - over) * c_1);
    }
  };
  row.visit([&](int col, float (&x)[4], int) {
    rest_of(x, col);
    const float big = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if constexpr (EPT > 0) {
      top[0] = fmaxf(top[0], big);
    } else {  // one reading for both: each thread's sums are over its own maximum so far
      if (big > top[0]) {
        sum[0] *= __builtin_amdgcn_exp2f((top[0] - big) * c_t);
        sum[1] *= __builtin_amdgcn_exp2f((top[0] - big) * c_1);
        top[0] = big;
      }
      add(x, top[0] == -INFINITY ? 0.f : top[0]);
    }
  });
  const float mine = top[0];
#pragma unroll
  DCR_ENTRIES(e) {
    top[1] = fmaxf(top[1], z_e[e]);
    top[2] = fmaxf(top[2], t_e[e]);
  }
  block_reduce_each<NT, 3>(top, red, MaxOp());
  const float mr = top[0], mk = top[1], mt = top[2], m = fmaxf(mr, mk);
  const float mr0 = mr == -INFINITY ? 0.f : mr;  // (an empty rest sums to 0)
  if constexpr (EPT > 0) {
    row.visit([&](int, float (&x)[4], int) { add(x, mr0); });
  } else if (mine > -INFINITY) {
    sum[0] *= __builtin_amdgcn_exp2f((mine - mr) * c_t);
    sum[1] *= __builtin_amdgcn_exp2f((mine - mr) * c_1);
  }
#pragma unroll
  DCR_ENTRIES(e) {
    if (first[e] && z_e[e] != -INFINITY) {
      sum[2] += expf(scaled(z_e[e] - mk, 0.f));
      if (two) sum[3] += expf(z_e[e] - mk);
    }
    if (t_e[e] != -INFINITY) sum[4] += expf(scaled(t_e[e] - mt, 0.f));
  }
  block_reduce_each<NT, 5>(sum, red + 3 * (NT / 64), AddOp());
  const float sr = sum[0], sr1 = two ? sum[1] : sum[0];
  const float sk = sum[2], sk1 = two ? sum[3] : sum[2];

  // a skipped row, and one whose mask leaves no column, has neither loss nor gradient
  const bool none = skip || (m == -INFINITY && sr == 0.f && sk == 0.f);
  // sums over m: no logit is scaled by itself, so the lowest values of the type stay finite
  const float dr = mr == -INFINITY ? -INFINITY : mr - m, dk = mk == -INFINITY ? -INFINITY : mk - m;
  const float wr = expf(scaled(dr, 0.f)), all = sr * wr + sk * expf(scaled(dk, 0.f));
  const float lse = logf(all), inv_all = 1.0f / all, off = sr * wr * inv_all;  // off: s
  const float wr1 = two ? expf(dr) : wr, all1 = two ? sr1 * wr1 + sk1 * expf(dk) : all;
  const bool told = a.lse != nullptr;
  const float tl = told ? a.lse[n] : 0.f;
  // entries that hold nothing say nothing, unless the teacher's mass lies elsewhere
  const bool mute = mt == -INFINITY && (!told || tl == -INFINITY);
  // log q = t / T - lt - log st, where without the teacher's log-sum-exp t counts from its maximum
  const float lt = told ? tl : logf(sum[4]), t0 = told ? 0.f : mt;
  float q_e[kE], p_e[kE], say[3] = {0.f, 0.f, 0.f};  // sums of q, of the terms, of q - p
#pragma unroll
  DCR_ENTRIES(e) {
    const float lq = t_e[e] != -INFINITY ? scaled(t_e[e] - t0, lt) : -INFINITY;
    const float d = lq - scaled(z_e[e] - m, lse);
    q_e[e] = expf(lq);
    p_e[e] = first[e] ? expf(scaled(z_e[e] - m, 0.f)) * inv_all : 0.f;
    if (i_e[e] < 0 || none) q_e[e] = p_e[e] = 0.f;
    say[0] += q_e[e];
    say[1] += q_e[e] <= 0.f ? p_e[e] : first[e] ? term(q_e[e], p_e[e], d) : q_e[e] * (d - 1.0f);
    say[2] += q_e[e] - p_e[e];
    if (e * NT + tid < k) eq[e * NT + tid] = q_e[e];
  }
  block_reduce_each<NT, 3>(say, red + 8 * (NT / 64), AddOp());
  if (NT == 64) __syncthreads();  // eq
  // what the teacher leaves (nothing where no column is left to hold it); the rest's gradient
  const float rest = told && mr > -INFINITY ? fmaxf(0.f, 1.0f - say[0]) : 0.f;
  float kl = say[1], pull = wr * inv_all;
  if (rest > 0.f) {
    float d;  // log(r / s)
    if (say[0] < 0.5f && fabsf(say[2]) <= 0.5f * off) {
      const float gap = say[2] / off;
      d = log1pf(-gap);
      pull *= gap;
    } else {
      // (s itself may be too small for a number)
      d = off > 1e-30f ? logf(rest / off) : logf(rest) - (scaled(dr, lse) + logf(sr));
      pull -= rest / sr;
    }
    kl += term(rest, off, d);
  } else {
    kl += off + (told ? say[0] - 1.0f : 0.f);
  }
  float loss = mute || a.alpha == 0.f ? 0.f : a.alpha_t2 * kl;
  if (ce) loss += (1.0f - a.alpha) * (logf(all1) - (z_y - m));
  if (tid == 0) a.row_loss[n] = none ? 0.f : loss;
  if (!grad) return;

  // ---- the gradient
  const float scale = a.scale * (a.gscale ? *a.gscale : 1.0f);
  const float ct = mute ? 0.f : a.alpha_t * scale, c1 = ce ? (1.0f - a.alpha) * scale : 0.f;
  // weights of exp((z - mr) / T) and exp(z - mr) off the entries
  float ft = ct == 0.f ? 0.f : ct * pull, f1 = c1 * wr1 / all1;
  if (mr == -INFINITY) ft = f1 = 0.f;
  if (!two) ft += f1, f1 = 0.f;
  if (none) ft = f1 = 0.f;
  // the target's chunk, for the thread that holds it
  const int cy = ce && !none && (y >> 2) % NT == tid ? (y >> 2) / NT : -1;
  row.visit([&](int col, float (&x)[4], int c) {
    const unsigned q = marked(col);
    rest_of(x, col);
    float g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = x[j] - mr0;
      g[j] = ft * __builtin_amdgcn_exp2f(d * c_t);
      if (two) g[j] += f1 * __builtin_amdgcn_exp2f(d * c_1);
    }
    if (c == cy)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((y & 3) == j) g[j] -= c1;
    if (none)
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = 0.f;
    if (q == 0 && col + 3 < V) {
      typename Vec4<G>::type o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (G)g[j];
      *reinterpret_cast<typename Vec4<G>::type*>(grad + col) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!(q >> j & 1) && col + j < V) grad[col + j] = (G)g[j];
    }
  });
#pragma unroll
  DCR_ENTRIES(e) {
    if (!first[e]) continue;
    float q = q_e[e];
    if (twice)
      for (int j = e * NT + tid + 1; j < k; ++j)
        if (ei[j] == i_e[e]) q += eq[j];
    float g = ct != 0.f ? ct * (p_e[e] - q) : 0.f;
    if (ce) g += c1 * expf(z_e[e] - m) / all1 - (i_e[e] == y ? c1 : 0.f);
    grad[i_e[e]] = (G)(none ? 0.f : g);
  }
}

#undef DCR_ENTRIES

// scale * sum of the row losses, in a fixed order
__global__ void __launch_bounds__(1024) distill_sum_kernel(const float* __restrict__ rows, int n,
                                                           float scale, float* __restrict__ out) {
  __shared__ float red[16];
  float s = 0.f;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 1024) s += rows[i];
  s = block_reduce<1024>(s, red, AddOp());
  if (threadIdx.x == 0) out[0] = s * scale;
}

// Workgroup and registers for N rows of V columns.  One wave takes a row of up to 1024 columns: no
// barriers, and many rows a CU.  Up to 16384 columns, few rows get more threads, which is faster for
// the row, and many get smaller workgroups, whose loads and computations overlap each other's.
// Launches of a replayed graph over two or three sets of rows, us, the larger workgroup against the
// smaller at 256, 512, 1024, 2048 and many rows:
//   1897 bf16 (256 threads, 64)            6.8  9.7    7.9 10.4   10.9 10.6   17.3 13.1   21294: 118 77
//   4000 fp32, two exponentials (256, 128) 7.9 10.3   10.0 13.1   15.2 15.1   23.0 22.2    8000: 67 63
//   8192 fp32 to bf16, two (512, 128)      9.1 16.3   14.5 21.3   22.5 24.6   37.7 38.6   32768: 464 355
//   12157 bf16 (512, 256)                 10.9 13.4   16.5 17.3   25.6 24.6   44.4 40.4    5296: 101 85
// (32768 x 8192 with 256 threads: 349.)  Past 32768 the registers are too few for two workgroups a CU,
// and a row is read twice instead (1024 x 65536 bf16: 99 us, 113 from registers; 2047 x 32001 bf16 112,
// 92 from registers).  Against the traffic at the rate of a large copy (5.0 TB/s): 32768 x 8192 322 us,
// 5296 x 12157 51, 21294 x 1897 32, 2047 x 32001 52.  What holds them is the issue of vector instructions:
// some 40 an element of 64 lanes, the units busy for 93 % of 2047 x 32001 and 98 % of 32768 x 8192.
template <typename T, typename G>
static void launch_types(const DistillArgs& a, hipStream_t s) {
  const size_t lds = (size_t)((a.r.V + 31) / 32) * 4;
  const int V = a.r.V;
  const bool many = a.r.N >= 1024;
#define CALL(NTH, E) distill_kernel<T, G, NTH, E><<<a.r.N, NTH, lds, s>>>(a)
  if (V <= 256) CALL(64, 4);
  else if (V <= 1024) CALL(64, 16);
  else if (V <= 2048 && many) CALL(64, 32);
  else if (V <= 4096 && many) CALL(128, 32);
  else if (V <= 4096) CALL(256, 16);
  else if (V <= 8192 && many) CALL(128, 64);
  else if (V <= 8192) CALL(512, 16);
  else if (V <= 16384 && many) CALL(256, 64);
  else if (V <= 16384) CALL(512, 32);
  else if (V <= 32768) CALL(512, 64);
  else CALL(1024, 0);
#undef CALL
}

void launch_distill(const DistillArgs& given, hipStream_t s) {
  DistillArgs a = given;
  const double inv = 1.0 / a.temperature;
  a.inv_t = (float)inv;
  a.inv_t_low = (float)(inv - (double)a.inv_t);
  a.log2e_t = (float)(1.4426950408889634 * inv);
  a.alpha_t = (float)(given.alpha * a.temperature);
  a.alpha_t2 = (float)(given.alpha * a.temperature * a.temperature);
  if (a.r.N > 0) {
    if (a.r.is_bf16) {
      if (a.grad_bf16) launch_types<bf16, bf16>(a, s); else launch_types<bf16, float>(a, s);
    } else {
      if (a.grad_bf16) launch_types<float, bf16>(a, s); else launch_types<float, float>(a, s);
    }
  }
  if (a.loss) distill_sum_kernel<<<1, 1024, 0, s>>>(a.row_loss, a.r.N, a.scale, a.loss);
}

}  // namespace dcr
