// Distillation from a teacher's recorded top logits: loss and gradient in one pass over the
// student's logits, beside the cross-entropy of xent.hip.
//
// With the student's p = softmax(z / T) and the teacher's recorded entries (i_j, t_j):
//   q_j = exp(t_j / T - lse), r = max(0, 1 - sum q_j)   with the teacher's log-sum-exp at T, or
//   q   = softmax_j(t_j / T), r = 0                     without it
//   loss = alpha T^2 [sum_j q_j (log q_j - log p_{i_j}) + r (log r - log s)]
//        + (1 - alpha) (lse(z) - z_y),                  s = the student's mass off the entries
//   d/dz_v = alpha T (p_v - q_v)            at the entries
//            alpha T p_v (1 - r / s)        elsewhere
//            + (1 - alpha) (softmax(z)_v - [v = y])
//
// One workgroup a row, the row in registers, so z is read once and the gradient written once:
// that traffic is the bound.  The recorded columns are marked in an LDS bitmap; their threads
// hold them apart (they write those gradients too), and the rest has a maximum and sum of its
// own.  So s is never a difference 1 - sum p, which has no digits left where the student is sure.
#include "vocab_row.h"

namespace dcr {

template <typename T, typename G, int NT, int EPT>
__global__ void __launch_bounds__(NT) distill_kernel(DistillArgs a) {
  extern __shared__ unsigned bits[];
  __shared__ float red[NT / 64];
  __shared__ float et[kRowMaxK], ez[kRowMaxK];  // entries: t / T, the student's z
  __shared__ int ei[kRowMaxK];                  // column; -1: no entry
  __shared__ unsigned char first[kRowMaxK];     // the first entry of its column
  __shared__ int twice;
  const long n = blockIdx.x;
  const int tid = threadIdx.x, V = a.r.V, k = a.k;
  const T* z = reinterpret_cast<const T*>(a.r.logits) + n * a.r.ld;
  G* grad = a.grad ? reinterpret_cast<G*>(a.grad) + n * a.grad_ld : nullptr;
  const float inv_t = 1.0f / a.temperature;
  const int y = a.targets ? a.targets[n] : 0;
  const bool skip = a.targets && (y < 0 || y >= V);
  const bool ce = a.targets && a.alpha < 1.0f;
  const bool two = ce && inv_t != 1.0f;  // a second exponential an element

  for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
  if (tid == 0) twice = 0;
  __syncthreads();
  for (int j = tid; j < k; j += NT) {
    const int i = a.indices[n * k + j];
    const bool ok = i >= 0 && i < V;
    ei[j] = ok ? i : -1;
    et[j] = ok ? a.values[n * k + j] * inv_t : -INFINITY;
    ez[j] = ok ? (float)z[i] : -INFINITY;
    first[j] = ok;
    if (ok && (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31) & 1)) twice = 1;
  }
  Row<T, NT, EPT> row(z, V);
  __syncthreads();
  if (twice) {  // a column recorded more than once: its first entry stands for it
    for (int j = tid; j < k; j += NT)
      for (int i = 0; i < j; ++i)
        if (ei[i] == ei[j]) first[j] = 0;
    __syncthreads();
  }
  // the entries' nibble of four columns
  auto marked = [&](int col) -> unsigned {
    return col < V ? bits[col >> 5] >> (col & 31) & 15u : 15u;
  };

  // ---- the rest: maximum, then the sums at T and at 1
  float mr = -INFINITY;
  row.visit([&](int col, float (&x)[4], int) {
    const unsigned q = marked(col);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(q >> j & 1)) mr = fmaxf(mr, x[j]);
  });
  mr = block_reduce<NT>(mr, red, MaxOp());
  float sr = 0.f, sr1 = 0.f;
  row.visit([&](int col, float (&x)[4], int) {
    const unsigned q = marked(col);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(q >> j & 1) && x[j] != -INFINITY) {
        sr += __expf((x[j] - mr) * inv_t);
        if (two) sr1 += __expf(x[j] - mr);
      }
  });
  sr = block_reduce<NT>(sr, red, AddOp());
  sr1 = two ? block_reduce<NT>(sr1, red, AddOp()) : sr;

  // ---- the entries
  float mk = -INFINITY, mt = -INFINITY;
  for (int j = tid; j < k; j += NT) {
    mk = fmaxf(mk, ez[j]);
    mt = fmaxf(mt, et[j]);
  }
  mk = block_reduce<NT>(mk, red, MaxOp());
  mt = block_reduce<NT>(mt, red, MaxOp());
  const float m = fmaxf(mr, mk);
  float sk = 0.f, sk1 = 0.f, st = 0.f;
  for (int j = tid; j < k; j += NT) {
    if (first[j] && ez[j] != -INFINITY) {
      sk += __expf((ez[j] - mk) * inv_t);
      if (two) sk1 += __expf(ez[j] - mk);
    }
    if (et[j] != -INFINITY) st += __expf(et[j] - mt);
  }
  sk = block_reduce<NT>(sk, red, AddOp());
  sk1 = two ? block_reduce<NT>(sk1, red, AddOp()) : sk;
  st = block_reduce<NT>(st, red, AddOp());

  // a skipped row, and one whose mask leaves no column, has neither loss nor gradient
  const bool none = skip || (m == -INFINITY && sr == 0.f && sk == 0.f);
  const float wr = mr == -INFINITY ? 0.f : __expf((mr - m) * inv_t);
  const float wk = mk == -INFINITY ? 0.f : __expf((mk - m) * inv_t);
  const float lse = m * inv_t + __logf(sr * wr + sk * wk);
  const float wr1 = mr == -INFINITY ? 0.f : __expf(mr - m);
  const float wk1 = mk == -INFINITY ? 0.f : __expf(mk - m);
  const float lse1 = m + __logf(sr1 * wr1 + sk1 * wk1);
  const bool told = a.lse != nullptr;
  // entries that hold nothing say nothing
  const float alpha = !told && mt == -INFINITY ? 0.f : a.alpha;
  const float lt = told ? a.lse[n] : mt + __logf(st);
  float sq = 0.f, kl = 0.f;
  for (int j = tid; j < k; j += NT)
    if (et[j] != -INFINITY) {
      const float lq = et[j] - lt, q = __expf(lq);
      sq += q;
      if (q > 0.f) kl += q * (lq - (ez[j] * inv_t - lse));
    }
  sq = block_reduce<NT>(sq, red, AddOp());
  kl = block_reduce<NT>(kl, red, AddOp());
  float rest = told ? fmaxf(0.f, 1.0f - sq) : 0.f;
  if (mr == -INFINITY) rest = 0.f;  // no column to hold it
  if (rest > 0.f) kl += rest * (__logf(rest) - (mr * inv_t + __logf(sr) - lse));
  float loss = alpha != 0.f ? alpha * a.temperature * a.temperature * kl : 0.f;
  if (ce) loss += (1.0f - a.alpha) * (lse1 - (float)z[skip ? 0 : y]);
  if (tid == 0) a.row_loss[n] = none ? 0.f : loss;
  if (!grad) return;

  // ---- the gradient
  const float scale = a.scale * (a.gscale ? *a.gscale : 1.0f);
  const float ct = alpha * a.temperature * scale, c1 = ce ? (1.0f - a.alpha) * scale : 0.f;
  // weights of exp((z - mr) / T) and exp(z - mr) off the entries
  const float ft = mr == -INFINITY ? 0.f
                                   : ct * (__expf(mr * inv_t - lse) - (rest > 0.f ? rest / sr : 0.f));
  const float f1 = mr == -INFINITY ? 0.f : c1 * __expf(mr - lse1);
  row.visit([&](int col, float (&x)[4], int) {
    const unsigned q = marked(col);
    float g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float e = 0.f;
      if (x[j] != -INFINITY) {
        const float et_ = __expf((x[j] - mr) * inv_t);
        e = ft * et_ + f1 * (two ? __expf(x[j] - mr) : et_);
      }
      if (ce && col + j == y) e -= c1;
      g[j] = none ? 0.f : e;
    }
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
  for (int j = tid; j < k; j += NT) {
    if (!first[j]) continue;
    float q = et[j] != -INFINITY ? __expf(et[j] - lt) : 0.f;
    if (twice)
      for (int i = j + 1; i < k; ++i)
        if (ei[i] == ei[j] && et[i] != -INFINITY) q += __expf(et[i] - lt);
    float e = ct != 0.f ? ct * (__expf(ez[j] * inv_t - lse) - q) : 0.f;
    if (ce) e += c1 * __expf(ez[j] - lse1) - (ei[j] == y ? c1 : 0.f);
    grad[ei[j]] = (G)(none ? 0.f : e);
  }
}

// scale * sum of the row losses, in a fixed order
__global__ void __launch_bounds__(1024) distill_sum_kernel(const float* __restrict__ rows, int n,
                                                           float scale, float* __restrict__ out) {
  __shared__ float red[16];
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += rows[i];
  s = block_reduce<1024>(s, red, AddOp());
  if (threadIdx.x == 0) out[0] = s * scale;
}

void launch_distill(const DistillArgs& a, hipStream_t s) {
  const size_t lds = (size_t)((a.r.V + 31) / 32) * 4;
#define CALL(NTH, E)                                                             \
  if (a.r.is_bf16) {                                                             \
    if (a.grad_bf16) distill_kernel<bf16, bf16, NTH, E><<<a.r.N, NTH, lds, s>>>(a); \
    else distill_kernel<bf16, float, NTH, E><<<a.r.N, NTH, lds, s>>>(a);         \
  } else {                                                                       \
    if (a.grad_bf16) distill_kernel<float, bf16, NTH, E><<<a.r.N, NTH, lds, s>>>(a); \
    else distill_kernel<float, float, NTH, E><<<a.r.N, NTH, lds, s>>>(a);        \
  }
  if (a.r.N > 0) DCR_ROW_DISPATCH(a.r.V, CALL);
#undef CALL
  if (a.loss) distill_sum_kernel<<<1, 1024, 0, s>>>(a.row_loss, a.r.N, a.scale, a.loss);
}

}  // namespace dcr
