// Gated linear recurrence over a sequence, forward and backward, for gfx950:
//
//   h_t = a_t h_{t-1} + s(-f_t) x_t,   a_t = s(f_t), or 0 where starts[t, b]   (s = logistic)
//
// and, with the gradients dh of the outputs and dlast of the final state,
//
//   g_t = dh_t + e_{t+1},  e_t = a_t g_t,   dx_t = s(-f_t) g_t,
//   df_t = s(f_t) s(-f_t) g_t (h_{t-1} or 0 at a start - x_t),   dh0 = e_0,   e_T = dlast.
//
// Steps t >= lengths[b] carry the state on (a = 1, no input), give output rows of zero and have
// no gradient.
//
// The step is linear in the state, so a stretch of steps is one pair (A, B): h_out = A h_in + B,
// and pairs combine.  A workgroup has 64 lanes x VEC channels (of the flattened [B, H]) and W
// waves; a tile is W x kC consecutive steps, kC a wave.  Each wave loads its steps once, forms
// its own pair in registers, the W pairs meet in LDS, and a second sweep over the registers
// writes the outputs: every element moves once in each direction, which is what bounds both
// kernels (2 reads + 1 write forward, 3 reads + 2 writes backward).  The forward leaves the fp32
// state in front of every tile (4 / (W kC) bytes per element); the backward recomputes the
// states of a tile from it in fp32, so it neither reads h nor sees h's rounding to bf16.
//
// 128 steps of 256 x 512 bf16: 22 us forward, 33 backward in a kernel trace over one set of inputs, which
// stays in the last-level cache in part, 26 and 42 over three sets in turn; the traffic takes 20 and 34 at
// the rate of a large copy (5.0 TB/s).
//
// Few channels and many steps leave too few workgroups: the time axis is then cut into
// segments, a first launch forms each segment's pair, and every workgroup of the second launch
// folds the pairs in front of its segment, in order, so the result does not depend on timing (every
// wave of it does, for itself).  16384 steps of 4 x 1000 bf16, padded documents, take some 385 us so, forward
// and backward; with x, f and dh read once each way the traffic would take 210.
#include "common.h"
#include "kernels.h"

namespace dcr {

namespace {

constexpr int kC = kLinrecSteps;

// wide loads at the alignment of one element: rows of odd width and offset views stay on them
template <typename T, int N>
struct VecOf;
template <int N>
struct VecOf<float, N> {
  typedef float type __attribute__((ext_vector_type(N), aligned(4)));
};
template <int N>
struct VecOf<bf16, N> {
  typedef bf16 type __attribute__((ext_vector_type(N), aligned(2)));
};

template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = (float)p[0];
  } else {
    const auto q = *reinterpret_cast<const typename VecOf<T, VEC>::type*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)q[j];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    p[0] = (T)v[0];
  } else {
    typename VecOf<T, VEC>::type q;
#pragma unroll
    for (int j = 0; j < VEC; ++j) q[j] = (T)v[j];
    *reinterpret_cast<typename VecOf<T, VEC>::type*>(p) = q;
  }
}

// s(f) and s(-f), both to full relative accuracy (1 - s(f) loses the small one)
__device__ __forceinline__ void gates(float f, float& keep, float& take) {
  const float t = __expf(-fabsf(f)), r = rcpf_(1.0f + t);
  keep = f >= 0.f ? r : t * r;
  take = f >= 0.f ? t * r : r;
}
// The factor of a stretch with a start: it lets nothing through, not even a NaN.  No product of gates
// is -0, so a product that is too small for a number stays apart from it, and a NaN state goes through
// that.  A lane's channels have their starts in common: the first one's factor is asked.
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float a) { return __float_as_uint(a) == 0x80000000u; }
// a h + b, or b where the stretch is cut
__device__ __forceinline__ float step_(bool cut, float a, float h, float b) {
  return cut ? b : __builtin_fmaf(a, h, b);
}

struct Lane {  // one lane's VEC channels
  bool on;
  int b, len;
  long c;  // flattened channel b * H + h
  int h;
};

// v through the pairs of n segments from `first` on, a batch of loads at a time (one after the other
// they would cost a cache's latency each).
template <bool MARKS, int VEC>
__device__ __forceinline__ void fold_pairs(float (&v)[VEC], const LinrecArgs& p, long c, int first,
                                           int dir, int n) {
  constexpr int kBatch = 16 / VEC;
  const long BH = (long)p.B * p.H;
  for (int s = 0; s < n; s += kBatch) {
    float A[kBatch][VEC], B[kBatch][VEC];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const long at = (first + dir * min(s + i, n - 1)) * BH + c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) A[i][j] = p.sumA[at + j], B[i][j] = p.sumB[at + j];
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (s + i < n) {
        const bool cut = MARKS && is_cut(A[i][0]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = step_(cut, A[i][j], v[j], B[i][j]);
      }
  }
}

// The second launch takes the segments the other way round: what the first read last is still
// in the last-level cache.
template <bool SUMMARY>
__device__ __forceinline__ int segment_of() {
  return SUMMARY ? blockIdx.y : gridDim.y - 1 - blockIdx.y;
}

template <int VEC>
__device__ __forceinline__ Lane lane_of(const LinrecArgs& p, int lane) {
  Lane l;
  const int HV = p.H / VEC;
  const long G = (long)p.B * HV;
  long g = (long)blockIdx.x * 64 + lane;
  l.on = g < G;
  if (!l.on) g = G - 1;  // the lane follows a valid one and stores nothing
  l.b = (int)(g / HV);
  l.h = (int)(g - (long)l.b * HV) * VEC;
  l.c = (long)l.b * p.H + l.h;
  l.len = p.lengths ? min(max(p.lengths[l.b], 0), p.T) : p.T;
  return l;
}

}  // namespace

// MARKS: lengths or starts are given.  SUMMARY: only the segment's pair (A, B) is formed
// (p.sumA / p.sumB).
template <typename T, int VEC, int W, bool MARKS, bool SUMMARY>
__global__ void __launch_bounds__(64 * W) linrec_fwd_kernel(LinrecArgs p) {
  __shared__ float sA[2][W][64 * VEC], sB[2][W][64 * VEC];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, seg = segment_of<SUMMARY>();
  const Lane l = lane_of<VEC>(p, lane);
  const T* x = reinterpret_cast<const T*>(p.x) + l.b * p.x_b + l.h;
  const T* f = reinterpret_cast<const T*>(p.f) + l.b * p.f_b + l.h;
  T* out = reinterpret_cast<T*>(p.h) + l.b * p.h_b + l.h;
  const unsigned char* st = p.starts ? p.starts + l.b * p.starts_b : nullptr;
  const long BH = (long)p.B * p.H;

  float carry[VEC], pa[VEC];  // the state in front of the tile; SUMMARY: the pair so far
  bool gone = false;          // SUMMARY: a start in it
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    carry[j] = (!SUMMARY && p.h0) ? p.h0[l.c + j] : 0.f;
    pa[j] = 1.f;
  }
  if (!SUMMARY) fold_pairs<MARKS, VEC>(carry, p, l.c, 0, 1, seg);

  const int tile1 = min((seg + 1) * p.tiles_per_seg, p.tiles);
  int buf = 0;
  for (int tile = seg * p.tiles_per_seg; tile < tile1; ++tile, buf ^= 1) {
    const int t0 = (tile * W + w) * kC;
    float a[kC][VEC], b[kC][VEC];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const long t = min(t0 + i, p.T - 1);
      load_row<T, VEC>(x + t * p.x_t, b[i]);
      load_row<T, VEC>(f + t * p.f_t, a[i]);
    }
    float A[VEC], B[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.f, B[j] = 0.f;
    bool cut = false;  // a start among the wave's steps
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const bool live = t0 + i < l.len;
      const bool start = MARKS && st && live && st[(long)(t0 + i) * p.starts_t];
      cut |= start;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float keep, take;
        gates(a[i][j], keep, take);
        a[i][j] = start ? kCut : live ? keep : 1.f;
        b[i][j] = live ? take * b[i][j] : 0.f;
        B[j] = step_(MARKS && is_cut(a[i][j]), a[i][j], B[j], b[i][j]);
        A[j] *= a[i][j];
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sA[buf][w][lane * VEC + j] = MARKS && cut ? kCut : A[j];
      sB[buf][w][lane * VEC + j] = B[j];
    }
    __syncthreads();  // (the other buffer's readers passed the previous tile's barrier)
    float h[VEC];
    if (!SUMMARY && p.carry && w == 0 && l.on)
#pragma unroll
      for (int j = 0; j < VEC; ++j) p.carry[tile * BH + l.c + j] = carry[j];
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[j] = carry[j];
#pragma unroll
    for (int ww = 0; ww < W; ++ww) {
      const bool none = MARKS && is_cut(sA[buf][ww][lane * VEC]);
      gone |= none;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (ww == w) h[j] = carry[j];
        const float aa = sA[buf][ww][lane * VEC + j];
        carry[j] = step_(none, aa, carry[j], sB[buf][ww][lane * VEC + j]);
        if (SUMMARY) pa[j] *= aa;
      }
    }
    if (!SUMMARY) {
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        float y[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          h[j] = step_(MARKS && is_cut(a[i][j]), a[i][j], h[j], b[i][j]);
          y[j] = t0 + i < l.len ? h[j] : 0.f;
        }
        if (l.on && t0 + i < p.T) store_row<T, VEC>(out + (long)(t0 + i) * p.h_t, y);
      }
    }
  }
  if (w == 0 && l.on) {
    if (SUMMARY) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        p.sumA[seg * BH + l.c + j] = gone ? kCut : pa[j];
        p.sumB[seg * BH + l.c + j] = carry[j];
      }
    } else if (seg == (int)gridDim.y - 1) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) p.hlast[l.c + j] = carry[j];
    }
  }
}

// Time runs backwards: e, the gradient with respect to the state in front of a stretch, is
// A e_out + G with the same A.  SUMMARY forms the segment's (A, G) from f and dh alone.
template <typename T, int VEC, int W, bool MARKS, bool SUMMARY>
__global__ void __launch_bounds__(64 * W) linrec_bwd_kernel(LinrecArgs p) {
  __shared__ float sA[2][W][64 * VEC], sB[2][W][64 * VEC], sG[2][W][64 * VEC];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, seg = segment_of<SUMMARY>();
  const Lane l = lane_of<VEC>(p, lane);
  const T* x = reinterpret_cast<const T*>(p.x) + l.b * p.x_b + l.h;
  const T* f = reinterpret_cast<const T*>(p.f) + l.b * p.f_b + l.h;
  const T* dh = reinterpret_cast<const T*>(p.dh) + l.b * p.dh_b + l.h;
  T* dx = reinterpret_cast<T*>(p.dx) + l.b * p.dx_b + l.h;
  T* df = reinterpret_cast<T*>(p.df) + l.b * p.df_b + l.h;
  const unsigned char* st = p.starts ? p.starts + l.b * p.starts_b : nullptr;
  const long BH = (long)p.B * p.H;

  float e[VEC], pa[VEC];  // the gradient behind the tile; SUMMARY: the pair so far
  bool gone = false;      // SUMMARY: a start in it
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    e[j] = (!SUMMARY && p.dlast) ? p.dlast[l.c + j] : 0.f;
    pa[j] = 1.f;
  }
  if (!SUMMARY)
    fold_pairs<MARKS, VEC>(e, p, l.c, (int)gridDim.y - 1, -1, (int)gridDim.y - 1 - seg);

  const int tile1 = min((seg + 1) * p.tiles_per_seg, p.tiles);
  int buf = 0;
  for (int tile = tile1 - 1; tile >= seg * p.tiles_per_seg; --tile, buf ^= 1) {
    const int t0 = (tile * W + w) * kC;
    float keep[kC][VEC], take[kC][VEC], xv[kC][VEC], g[kC][VEC];
    unsigned cut = 0;  // bit i: step t0 + i is a start
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const long t = min(t0 + i, p.T - 1);
      if (!SUMMARY) load_row<T, VEC>(x + t * p.x_t, xv[i]);
      load_row<T, VEC>(f + t * p.f_t, keep[i]);
      load_row<T, VEC>(dh + t * p.dh_t, g[i]);
    }
    float A[VEC], B[VEC], G[VEC], h[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.f, B[j] = 0.f, G[j] = 0.f;
    if (!SUMMARY)
#pragma unroll
      for (int j = 0; j < VEC; ++j) h[j] = p.carry[tile * BH + l.c + j];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      const bool live = t0 + i < l.len;
      if (MARKS && st && live && st[(long)(t0 + i) * p.starts_t]) cut |= 1u << i;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        gates(keep[i][j], keep[i][j], take[i][j]);
        if (!live) keep[i][j] = 1.f, take[i][j] = 0.f, g[i][j] = 0.f;
        if (!live && !SUMMARY) xv[i][j] = 0.f;
        if (SUMMARY) {
          A[j] *= keep[i][j];
        } else {
          const float a = MARKS && (cut >> i & 1) ? kCut : keep[i][j];
          B[j] = step_(MARKS && is_cut(a), a, B[j], take[i][j] * xv[i][j]);
          A[j] *= a;
        }
      }
    }
#pragma unroll
    for (int i = kC - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        G[j] = (MARKS && (cut >> i & 1)) ? 0.f : keep[i][j] * (g[i][j] + G[j]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sA[buf][w][lane * VEC + j] = MARKS && cut ? kCut : A[j];
      sG[buf][w][lane * VEC + j] = G[j];
      if (!SUMMARY) sB[buf][w][lane * VEC + j] = B[j];
    }
    __syncthreads();
    if (!SUMMARY)
#pragma unroll
      for (int ww = 0; ww < W - 1; ++ww)
        if (ww < w) {
          const bool none = MARKS && is_cut(sA[buf][ww][lane * VEC]);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            h[j] = step_(none, sA[buf][ww][lane * VEC + j], h[j], sB[buf][ww][lane * VEC + j]);
        }
    float ein[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) ein[j] = e[j];
#pragma unroll
    for (int ww = W - 1; ww >= 0; --ww) {
      const bool none = MARKS && is_cut(sA[buf][ww][lane * VEC]);
      gone |= none;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (ww == w) ein[j] = e[j];
        const float aa = sA[buf][ww][lane * VEC + j];
        e[j] = step_(none, aa, e[j], sG[buf][ww][lane * VEC + j]);
        if (SUMMARY) pa[j] *= aa;
      }
    }
    if (!SUMMARY) {
      float hp[kC][VEC];  // the state that step i multiplies
#pragma unroll
      for (int i = 0; i < kC; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          hp[i][j] = (MARKS && (cut >> i & 1)) ? 0.f : h[j];
          h[j] = __builtin_fmaf(keep[i][j], hp[i][j], take[i][j] * xv[i][j]);
        }
#pragma unroll
      for (int i = kC - 1; i >= 0; --i) {
        float ox[VEC], of[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float gi = g[i][j] + ein[j];
          const float cg = take[i][j] * gi;
          ox[j] = t0 + i < l.len ? cg : 0.f;
          of[j] = t0 + i < l.len ? keep[i][j] * cg * (hp[i][j] - xv[i][j]) : 0.f;
          ein[j] = (MARKS && (cut >> i & 1)) ? 0.f : keep[i][j] * gi;
        }
        if (l.on && t0 + i < p.T) {
          store_row<T, VEC>(dx + (long)(t0 + i) * p.dx_t, ox);
          store_row<T, VEC>(df + (long)(t0 + i) * p.df_t, of);
        }
      }
    }
  }
  if (w == 0 && l.on) {
    if (SUMMARY) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        p.sumA[seg * BH + l.c + j] = gone ? kCut : pa[j];
        p.sumB[seg * BH + l.c + j] = e[j];
      }
    } else if (seg == 0 && p.dh0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) p.dh0[l.c + j] = e[j];
    }
  }
}

// One step of every stream: the fp32 state in place, the output in the inputs' type.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) linrec_step_kernel(LinrecArgs p) {
  const int HV = p.H / VEC;
  const long g = (long)blockIdx.x * 256 + threadIdx.x;
  if (g >= (long)p.B * HV) return;
  const int b = (int)(g / HV), hh = (int)(g - (long)b * HV) * VEC;
  float x[VEC], f[VEC], h[VEC];
  load_row<T, VEC>(reinterpret_cast<const T*>(p.x) + b * p.x_b + hh, x);
  load_row<T, VEC>(reinterpret_cast<const T*>(p.f) + b * p.f_b + hh, f);
  float* hs = p.hlast + (long)b * p.H + hh;
  load_row<float, VEC>(hs, h);
  const bool start = p.starts && p.starts[b * p.starts_b];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    float keep, take;
    gates(f[j], keep, take);
    h[j] = start ? take * x[j] : __builtin_fmaf(keep, h[j], take * x[j]);
  }
  store_row<float, VEC>(hs, h);
  store_row<T, VEC>(reinterpret_cast<T*>(p.h) + b * p.h_b + hh, h);
}

namespace {

template <typename T, int VEC, int W, bool MARKS>
void run_seq(LinrecArgs& p, bool bwd, hipStream_t s) {
  const long groups = (long)p.B * (p.H / VEC);
  const dim3 grid((unsigned)((groups + 63) / 64), (unsigned)p.segs), block(64 * W);
  if (bwd) {
    if (p.segs > 1) linrec_bwd_kernel<T, VEC, W, MARKS, true><<<grid, block, 0, s>>>(p);
    linrec_bwd_kernel<T, VEC, W, MARKS, false><<<grid, block, 0, s>>>(p);
  } else {
    if (p.segs > 1) linrec_fwd_kernel<T, VEC, W, MARKS, true><<<grid, block, 0, s>>>(p);
    linrec_fwd_kernel<T, VEC, W, MARKS, false><<<grid, block, 0, s>>>(p);
  }
}

template <typename T, int W>
void run_type(LinrecArgs& p, bool bwd, int vec, hipStream_t s) {
  const bool marks = p.lengths || p.starts;
#define LR(VV) \
  if (marks) run_seq<T, VV, W, true>(p, bwd, s); else run_seq<T, VV, W, false>(p, bwd, s)
  if constexpr (W <= 4) {
    if (vec == 4) {
      LR(4);
      return;
    }
  }
  if (vec == 2) { LR(2); } else { LR(1); }
#undef LR
}

}  // namespace

// Channels a lane, waves a workgroup and segments of the time axis, from the sizes and the type alone
// (the backward has to find the forward's tiles).  Measured on one MI355X, launches of a replayed graph
// over three sets of inputs, forward / backward us:
//  * the widest loads that leave some 192 workgroups, else single channels: 25600 channels, 1024
//    steps, bf16: 52 / 71 with two channels a lane, 56 / 78 with one, 101 / 124 with four; 12800 channels,
//    200 steps: 10.1 / 12.9 with one, 12.6 / 16.1 with two;
//  * no more waves than the steps fill (8 steps of 256 x 2048 bf16: 9.4 / 12.1 with one, 15.5 / 24.9
//    with four); then four waves where a lane has four channels (128 steps of 256 x 512 bf16: 26 / 42,
//    with eight 26 / 47; 16384 steps of 4 x 1000, padded documents: 167 / 231 against 180 / 253), else
//    eight: longer tiles, fewer of them (4096 steps of 512 channels: 13.1 / 20.3, with four 14.9 / 23.8);
//  * segments where there are few workgroups of single channels and many steps, although x, f and dh
//    are then read twice (4096 steps of 512 channels: 13.1 / 20.3 with 64 segments, 18 / 35 with 16; 200
//    steps of 6400 channels: one segment 8.5 / 12.1, four 12.9 / 16.3).  Both directions together, in
//    segments against one: 512 steps, 48 workgroups 27 against 36 bf16, 26 against 37 fp32; 94: 45
//    against 39, 37 against 37; 191: 53 against 39, 66 against 51.  768 steps, 94: 51 against 54, 60
//    against 58; 157: 55 against 54, 79 against 71.  1000 steps, 125: 56 against 69, 82 against 88;
//    157: 70 against 74, 112 against 93; 191: 81 against 76, 128 against 97.  4096 steps, 125: 181
//    against 300, 336 against 331; 157: 236 against 307, 438 against 348.  At most 128 (15390 steps of
//    384 channels bf16: 71, with at most 64 78): each workgroup folds the pairs in front of its segment.
LinrecPlan linrec_plan(int T, int B, int H, bool is_bf16) {
  LinrecPlan q{};
  auto wgs = [&](int vec) { return ((long)B * (H / vec) + 63) / 64; };
  const int widest = H % 4 == 0 ? 4 : H % 2 == 0 ? 2 : 1;
  const bool split = T >= 512 && wgs(1) * 6 < T && wgs(1) < (is_bf16 ? 192 : 128);
  const long cuts = split ? (T / 64 < 128 ? T / 64 : 128) : 1;
  q.vec = widest;
  while (q.vec > 1 && wgs(q.vec) * cuts < (split ? 512 : 192)) q.vec /= 2;
  const long n = wgs(q.vec) > 0 ? wgs(q.vec) : 1;
  q.waves = T <= kC ? 1 : T <= 2 * kC ? 2 : T <= 4 * kC || q.vec == 4 ? 4 : 8;
  q.tiles = (T + q.waves * kC - 1) / (q.waves * kC);
  long segs = split ? ((q.waves == 4 ? 1024 : 512) + n - 1) / n : 1;
  if (segs > 128) segs = 128;
  q.tiles_per_seg = (int)((q.tiles + segs - 1) / segs);
  if (q.tiles_per_seg < 1) q.tiles_per_seg = 1;
  q.segs = (q.tiles + q.tiles_per_seg - 1) / q.tiles_per_seg;
  if (q.segs < 1) q.segs = 1;
  return q;
}

void launch_linrec(LinrecArgs p, bool is_bf16, bool bwd, hipStream_t s) {
  const LinrecPlan q = linrec_plan(p.T, p.B, p.H, is_bf16);
  p.tiles = q.tiles;
  p.tiles_per_seg = q.tiles_per_seg;
  p.segs = q.segs;
#define LW(WW) \
  if (is_bf16) run_type<bf16, WW>(p, bwd, q.vec, s); else run_type<float, WW>(p, bwd, q.vec, s)
  if (q.waves == 1) { LW(1); } else if (q.waves == 2) { LW(2); }
  else if (q.waves == 4) { LW(4); } else { LW(8); }
#undef LW
}

void launch_linrec_step(const LinrecArgs& p, bool is_bf16, hipStream_t s) {
  const int vec = p.H % 4 == 0 ? 4 : p.H % 2 == 0 ? 2 : 1;
  const unsigned nb = (unsigned)(((long)p.B * (p.H / vec) + 255) / 256);
#define LS(TT, VV) linrec_step_kernel<TT, VV><<<nb, 256, 0, s>>>(p)
  if (is_bf16) {
    if (vec == 4) LS(bf16, 4); else if (vec == 2) LS(bf16, 2); else LS(bf16, 1);
  } else {
    if (vec == 4) LS(float, 4); else if (vec == 2) LS(float, 2); else LS(float, 1);
  }
#undef LS
}

}  // namespace dcr
