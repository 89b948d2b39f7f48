// Losses and records over rows of vocabulary logits (gfx950).
//
// A row is x in R^V with V from a few hundred to a few hundred thousand. With
// M = max x, S = sum exp((x-M)/t), q_j = exp((x_j-M)/t) / S and
// log q_j = (x_j-M)/t - log S, everything here is one of
//
//   stats   one pass over x for (M, S), a running maximum and sum per thread
//   finish  one thread per row: the loss from (M, S) and a few gathered logits,
//           and the coefficients of its gradient
//   grad    one pass over x that writes dx_j = a (q_j - p_j), p_j != 0 in K places
//
// All three are bound by memory: stats reads x, grad reads x and writes dx, so
// a training step moves 3 * V * sizeof(T) per row. (x - M) is taken before the
// product with log2(e)/t: exact for logits near M, and the type's lowest value
// as a mask neither overflows nor, where a whole row holds it, gives a NaN.
// Sums of exponentials are held in 32 bits per thread, joined in 32, and every
// logarithm, divergence and sum over rows is taken in 64.
#include "common.h"
#include "lm_loss.h"

#include <cfloat>

namespace {

constexpr int kThreads = 256;
constexpr double kLog2e = 1.4426950408889634074;

// 16 bytes at the alignment of one element: rows of an odd V start anywhere.
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
typedef float f32x8_v __attribute__((ext_vector_type(8)));

template <int TY>
struct Ty;
template <>
struct Ty<LM_BF16> {
  static constexpr int N = 8, size = 2, low_bits = 16;
  static DEVINL float one(const char* p) { return bf16_to_f32(*(const short*)p); }
  static DEVINL void put(char* p, float v) { *(__bf16*)p = (__bf16)v; }
  static DEVINL void open(u32x4 r, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(r[i] << 16);
      f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
  static DEVINL u32x4 close(const float* f) {
    f32x8_v v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i];
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8_v));
  }
};
template <>
struct Ty<LM_FP16> {
  static constexpr int N = 8, size = 2, low_bits = 13;
  static DEVINL float one(const char* p) { return (float)*(const _Float16*)p; }
  static DEVINL void put(char* p, float v) { *(_Float16*)p = (_Float16)v; }
  static DEVINL void open(u32x4 r, float* f) {
    f16x8_v h = __builtin_bit_cast(f16x8_v, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  }
  static DEVINL u32x4 close(const float* f) {
    f32x8_v v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i];
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8_v));
  }
};
template <>
struct Ty<LM_FP32> {
  static constexpr int N = 4, size = 4, low_bits = 0;
  static DEVINL float one(const char* p) { return *(const float*)p; }
  static DEVINL void put(char* p, float v) { *(float*)p = v; }
  static DEVINL void open(u32x4 r, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r[i]);
  }
  static DEVINL u32x4 close(const float* f) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(f[i]);
    return r;
  }
};

DEVINL float one_of(int type, const char* base, long long i) {
  return type == LM_BF16   ? Ty<LM_BF16>::one(base + i * 2)
         : type == LM_FP16 ? Ty<LM_FP16>::one(base + i * 2)
                           : Ty<LM_FP32>::one(base + i * 4);
}

DEVINL long long row_start(const LmRows& in, int r) {
  int b = r / in.T;
  return (long long)b * in.sb + (long long)(r - b * in.T) * in.st;
}

DEVINL long long place(const LmPlaces& pl, long long i) {
  return pl.idx64 ? ((const long long*)pl.idx)[i]
                  : (long long)((const int*)pl.idx)[i];
}

DEVINL bool ignored(const LmPlaces& pl, int r) {
  return (pl.mask && !pl.mask[r]) ||
         (pl.use_ignore && place(pl, r) == pl.ignore);
}

// 2^a by the hardware instruction: results under 2^-126 are 0, which changes
// no sum that has a term of 1 and no probability that a float can tell from 0.
DEVINL float exp2_hw(float a) { return __builtin_amdgcn_exp2f(a); }

// 2^(d log2(e)/t) with the constant in two parts: one float of it is off by up
// to 2^-25, the same way for every logit, and that would be 1e-7 in log S, in
// one direction for all the tokens of an answer.
DEVINL float exp_of(float d, const LmRows& in) {
  return exp2_hw(fmaf(d, in.c, d * in.c_lo));
}

// A running maximum and the sum of 2^((x-m)c) below it. m starts at the least
// finite float, so that -inf adds 0 and never meets itself in a difference.
struct Run {
  float m, s;
  DEVINL void join(float om, float os, float c) {
    float mn = fmaxf(m, om);
    s = s * exp2_hw((m - mn) * c) + os * exp2_hw((om - mn) * c);
    m = mn;
  }
};
DEVINL Run run_empty() { return {-FLT_MAX, 0.f}; }

template <int THREADS>
DEVINL Run block_join(Run a, float c, Run* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    float om = __shfl_xor(a.m, off, 64), os = __shfl_xor(a.s, off, 64);
    a.join(om, os, c);
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) a.join(red[w].m, red[w].s, c);
  return a;
}

DEVINL double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// the sum over a block in every thread, in one order
DEVINL double block_sum(double v, double* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) v += red[w];
  return v;
}

// A record's probabilities by one block, K <= 256, in 64 bits as 1 - sum p
// follows. rec = {sum p log p, sum p x, sum p, rest}, rest < 0 marks a row
// without a record.
DEVINL void record_of(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
                      int r, float* p_out, double4* rec) {
  __shared__ double red[kThreads / 64];
  __shared__ float mred[kThreads / 64];
  const int k = threadIdx.x;
  const long long at = (long long)r * pl.K + k;
  const long long j = k < pl.K ? place(pl, at) : -1;
  const float v = j >= 0 ? one_of(te.type, (const char*)te.values, at) : -INFINITY;
  const bool some = v > -INFINITY || v != v;
  if (__syncthreads_count(some) == 0) {
    if (k == 0) rec[r] = make_double4(0, 0, 0, -1);
    return;
  }
  const double t = te.temperature;
  double lp;
  if (te.lse) {
    lp = (double)v / t - te.lse[r];
  } else {
    float m = v;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if ((k & 63) == 0) mred[k >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(mred[0], mred[1]), fmaxf(mred[2], mred[3]));
    lp = ((double)v - m) / t;
    lp -= log(block_sum(some ? exp(lp) : 0.0, red));
  }
  double p = some ? exp(lp) : 0.0, x = 0.0;
  if (p != 0.0) {
    x = j < in.V ? (double)one_of(in.type, (const char*)in.x, row_start(in, r) + j)
                 : NAN;
    if (j >= in.V) p = NAN;
  }
  const double a = block_sum(p != 0.0 ? p * lp : 0.0, red);
  const double b = block_sum(p != 0.0 ? p * x : 0.0, red);
  const double sum = block_sum(p, red);
  if (k < pl.K) p_out[at] = (float)p;
  if (k == 0)
    rec[r] = make_double4(a, b, sum, te.lse ? fmax(1.0 - sum, 0.0) : 0.0);
}

// ------------------------------------------------------------------- stats
// grid R*splits, block (r, s) takes `seg` logits from s*seg on; R more blocks,
// the first ones, make the records of a distillation. With TOP, the
// K places of a record are kept apart: a bit per logit of the segment in LDS,
// so that the sum outside the record is one of its own and not the difference
// of two that nearly cancel.
template <int TY, bool TOP>
__global__ void __launch_bounds__(kThreads)
    lm_stats_kernel(LmRows in, LmPlaces pl, LmTeacher te, int splits, int seg,
                    float2* __restrict__ part, float2* __restrict__ part_top,
                    float* __restrict__ p, double4* __restrict__ rec,
                    int* __restrict__ counter) {
  using X = Ty<TY>;
  extern __shared__ unsigned bits[];
  __shared__ Run red[kThreads / 64];
  const int tid = threadIdx.x;
  if (blockIdx.x == 0 && tid == 0) *counter = 0;  // for the finish kernel
  int at_block = blockIdx.x;
  if (te.values) {
    if (at_block < in.R) {
      if (!ignored(pl, at_block)) record_of(in, pl, te, at_block, p, rec);
      return;
    }
    at_block -= in.R;
  }
  const int r = at_block / splits, sp = at_block - r * splits;
  if (ignored(pl, r)) return;
  const int v0 = sp * seg;
  const int n = min(seg, in.V - v0);
  const char* x = (const char*)in.x + (row_start(in, r) + v0) * X::size;
  const float c = in.c;
  const int nv = n / X::N;
  if (TOP) {
    for (int i = tid; i < (n + 31) / 32; i += kThreads) bits[i] = 0;
    __syncthreads();
    for (int k = tid; k < pl.K; k += kThreads) {
      long long j = place(pl, (long long)r * pl.K + k) - v0;
      if (j >= 0 && j < n) atomicOr(&bits[j >> 5], 1u << (j & 31));
    }
    __syncthreads();
  }
  Run a = run_empty(), top = run_empty();
  constexpr int Q = 4;  // 16-byte loads in flight per thread
  for (int i = tid; i < nv; i += Q * kThreads) {
    float f[Q * X::N];
#pragma unroll
    for (int g = 0; g < Q; ++g) {
      const int ig = i + g * kThreads;
      if (ig < nv) {
        X::open(*(const u32x4_any*)(x + (long long)ig * 16), f + g * X::N);
      } else {
#pragma unroll
        for (int e = 0; e < X::N; ++e) f[g * X::N + e] = -INFINITY;
      }
    }
    if (TOP) {
#pragma unroll
      for (int g = 0; g < Q; ++g) {
        const int j = (i + g * kThreads) * X::N;
        unsigned hit = j < n ? bits[j >> 5] >> (j & 31) : 0u;
        hit &= (1u << X::N) - 1u;
        if (hit) {
#pragma unroll
          for (int e = 0; e < X::N; ++e)
            if (hit >> e & 1) {
              top.join(f[g * X::N + e], 1.f, c);
              f[g * X::N + e] = -INFINITY;
            }
        }
      }
    }
    float vm = a.m;
#pragma unroll
    for (int e = 0; e < Q * X::N; ++e) vm = fmaxf(vm, f[e]);
    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < Q * X::N; ++e) add[e & 3] += exp_of(f[e] - vm, in);
    a.s = a.s * exp_of(a.m - vm, in) + ((add[0] + add[1]) + (add[2] + add[3]));
    a.m = vm;
  }
  if (tid < n - nv * X::N) {  // what is left of a vector
    int j = nv * X::N + tid;
    float f = X::one(x + (long long)j * X::size);
    if (TOP && (bits[j >> 5] >> (j & 31) & 1))
      top.join(f, 1.f, c);
    else
      a.join(f, 1.f, c);
  }
  a = block_join<kThreads>(a, c, red);
  if (TOP) {
    __syncthreads();
    top = block_join<kThreads>(top, c, red);
  }
  if (tid == 0) {
    long long at = (long long)sp * in.R + r;
    part[at] = make_float2(a.m, a.s);
    if (TOP) part_top[at] = make_float2(top.m, top.s);
  }
}

// the splits of a row as one, in 64 bits from here on
struct Row {
  double m, s;
};
DEVINL Row join_splits(const float2* part, int splits, int R, int r, double c) {
  float m = -FLT_MAX;
  for (int i = 0; i < splits; ++i) m = fmaxf(m, part[(long long)i * R + r].x);
  double s = 0.0;
  for (int i = 0; i < splits; ++i) {
    float2 q = part[(long long)i * R + r];
    s += q.x == m ? (double)q.y : (double)q.y * exp2(((double)q.x - m) * c);
  }
  return {(double)m, s};
}

// Sum of `loss` and `count` over the whole grid, in one order: each block's
// sums in memory, the block that arrives last adds them up. *o.loss = the loss,
// *o.inv = 1/count for a mean over the rows that count, else 1.
DEVINL void grid_mean(double loss, double count, double2* bpart, int* counter,
                      const LmOut& o) {
  __shared__ double red[16];
  __shared__ int last;
  loss = block_sum(loss, red);
  count = block_sum(count, red);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      bpart[blockIdx.x] = make_double2(loss, count);
      __threadfence();
      last = atomicAdd(counter, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    loss = count = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += blockDim.x) {
      loss += __hip_atomic_load(&bpart[i].x, __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_AGENT);
      count += __hip_atomic_load(&bpart[i].y, __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_AGENT);
    }
    loss = block_sum(loss, red);
    count = block_sum(count, red);
  }
  if (threadIdx.x == 0) {
    const double inv = o.reduction == LM_MEAN ? 1.0 / fmax(count, 1.0) : 1.0;
    *o.loss = (float)(loss * inv);
    *o.inv = (float)inv;
  }
}

// ------------------------------------------------------------------ distill
__global__ void __launch_bounds__(kThreads)
    lm_distill_kernel(LmRows in, LmPlaces pl, LmTeacher te, int splits,
                      const float2* __restrict__ part,
                      const float2* __restrict__ part_top,
                      const double4* __restrict__ rec,
                      LmStat* __restrict__ stat, float* __restrict__ coef,
                      double2* bpart, int* counter, LmOut o) {
  const int r = blockIdx.x * kThreads + threadIdx.x;
  double loss = 0.0, count = 0.0;
  if (r < in.R) {
    LmStat st = {0.f, 0.f, 0.f, 0.f};
    float a = 0.f;
    const bool live = !ignored(pl, r);
    const double4 k = live ? rec[r] : make_double4(0, 0, 0, -1);
    if (live && !(k.w < 0.0)) {
      const double t = te.temperature, c = kLog2e / t;
      Row rest = join_splits(part, splits, in.R, r, c), all = rest;
      // dL/dx_j t = mass q_j - p_j, mass = sum p + rest: 1, if the record's
      // values and its logsumexp are of the same row
      double tail = 0.0, mass = k.z;
      if (te.lse) {
        Row top = join_splits(part_top, splits, in.R, r, c);
        all.m = fmax(rest.m, top.m);
        double sr = rest.s * exp((rest.m - all.m) / t);
        all.s = sr + top.s * exp((top.m - all.m) / t);
        // no logit outside the record is above -inf: it has no rest
        if (rest.s != 0.0) {
          double log_rest = (rest.m - all.m) / t + log(rest.s / all.s);
          if (k.w > 0.0) tail = k.w * (log(k.w) - log_rest);
          mass += k.w;
          st.w = (float)((mass * exp(log_rest) - k.w) / rest.s);
        }
      } else {
        st.w = (float)(mass / all.s);
      }
      st.mb = (float)rest.m;
      st.M = (float)all.m;
      st.mass_S = (float)(mass / all.s);
      loss = k.x - (k.y - k.z * all.m) / t + k.z * log(all.s) + tail;
      loss *= t * t;
      count = 1.0;
      // d/dx of t^2 KL(x/t); a NaN, of a place outside the row too, is the
      // whole row's
      a = loss == loss ? (float)t : NAN;
    }
    stat[r] = st;
    coef[r] = a;
    if (o.reduction == LM_NONE) o.loss[r] = (float)loss;
  }
  if (o.reduction != LM_NONE) grid_mean(loss, count, bpart, counter, o);
}

// ------------------------------------------- log-probability of one token
// lp = (x_t - M) - log S; a target outside the row gives NaN
DEVINL double token_logp(const LmRows& in, const LmPlaces& pl, int r, int splits,
                         const float2* part, LmStat* st) {
  Row a = join_splits(part, splits, in.R, r, kLog2e);
  long long j = place(pl, r);
  double x = j >= 0 && j < in.V
                 ? (double)one_of(in.type, (const char*)in.x, row_start(in, r) + j)
                 : NAN;
  float inv = (float)(1.0 / a.s);
  *st = {(float)a.m, inv, (float)a.m, inv};
  return (x - a.m) - log(a.s);
}

__global__ void __launch_bounds__(kThreads)
    lm_policy_kernel(LmRows in, LmPlaces pl, LmPolicy po, int splits,
                     const float2* __restrict__ part, LmStat* __restrict__ stat,
                     float* __restrict__ coef, float* __restrict__ logps,
                     float* __restrict__ kls, double2* bpart, int* counter,
                     LmOut o) {
  const int r = blockIdx.x * kThreads + threadIdx.x;
  double loss = 0.0, count = 0.0;
  if (r < in.R) {
    LmStat st = {0.f, 0.f, 0.f, 0.f};
    double by_lp = 0.0, lp = 0.0, kl = 0.0;
    if (!ignored(pl, r)) {
      lp = token_logp(in, pl, r, splits, part, &st);
      const double A = po.adv[r], lo = 1.0 - po.clip_low,
                   hi = 1.0 + po.clip_high;
      const double ratio = exp(lp - (double)po.old_lp[r]);
      const double held = fmin(fmax(ratio, lo), hi);
      // the lesser of ratio*A and held*A; a NaN stays one
      const bool moves = A > 0.0 ? !(ratio > hi) : !(ratio < lo);
      loss = moves ? -ratio * A : -held * A;
      by_lp = moves ? -ratio * A : 0.0;
      if (po.ref_lp) {
        const double d = (double)po.ref_lp[r] - lp, e = expm1(d);
        kl = e - d;
        loss += po.kl_coef * kl;
        by_lp -= po.kl_coef * e;
      }
      count = 1.0;
    }
    stat[r] = st;
    // the gradient is coef * (q - onehot)
    coef[r] = (float)-by_lp;
    logps[r] = (float)lp;
    kls[r] = (float)kl;
    if (o.reduction == LM_NONE) o.loss[r] = (float)loss;
  }
  if (o.reduction != LM_NONE) grid_mean(loss, count, bpart, counter, o);
}

// One block per pair: sequences n and n + N. The sums over an answer are held
// in 64 bits, as the loss is made of the small differences between them.
__global__ void __launch_bounds__(1024)
    lm_preference_kernel(LmRows in, LmPlaces pl, LmPreference pr, int splits,
                         const float2* __restrict__ part,
                         LmStat* __restrict__ stat, float* __restrict__ coef,
                         float* __restrict__ chosen,
                         float* __restrict__ rejected, double2* bpart,
                         int* counter, LmOut o) {
  __shared__ double red[16];
  const int n = blockIdx.x, N = gridDim.x, T = in.T;
  double sum[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    double part_sum = 0.0;
    const int r0 = (n + side * N) * T;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
      LmStat st = {0.f, 0.f, 0.f, 0.f};
      if (!ignored(pl, r0 + t))
        part_sum += token_logp(in, pl, r0 + t, splits, part, &st);
      stat[r0 + t] = st;
    }
    sum[side] = block_sum(part_sum, red);
  }
  double reward[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int b = n + side * N;
    const double ref = pr.ref64 ? ((const double*)pr.ref)[b]
                                : (double)((const float*)pr.ref)[b];
    reward[side] = pr.beta * (sum[side] - ref);
  }
  const double z = reward[0] - reward[1], e = pr.smoothing;
  const double softplus = fmax(z, 0.0) + log1p(exp(-fabs(z)));
  double loss = (1.0 - e) * (softplus - z) + e * softplus;
  if (z != z) loss = z;
  const double by_z = 1.0 / (1.0 + exp(-z)) - (1.0 - e);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int r0 = (n + side * N) * T;
    const float a = (float)((side ? 1.0 : -1.0) * pr.beta * by_z);
    for (int t = threadIdx.x; t < T; t += blockDim.x)
      coef[r0 + t] = ignored(pl, r0 + t) ? 0.f : a;
  }
  if (threadIdx.x == 0) {
    chosen[n] = (float)reward[0];
    rejected[n] = (float)reward[1];
    if (o.reduction == LM_NONE) o.loss[n] = (float)loss;
  }
  if (o.reduction != LM_NONE)
    grid_mean(threadIdx.x == 0 ? loss : 0.0, threadIdx.x == 0 ? 1.0 : 0.0,
              bpart, counter, o);
}

// --------------------------------------------------------------------- grad
// grid R*splits; block (r, s) reads its segment and writes the gradient. A row
// whose coefficient is 0 (ignored, or clipped) is not read. The rows go from
// the last to the first, as the last ones that stats read are the likeliest
// to be still in the cache.
template <int TY, bool ONE>
__global__ void __launch_bounds__(kThreads)
    lm_grad_kernel(LmRows in, LmPlaces pl, LmKeep kp, LmUp up,
                   char* __restrict__ dx_all, int splits, int seg) {
  using X = Ty<TY>;
  __shared__ long long s_idx[kThreads];
  __shared__ float s_p[kThreads];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / splits, sp = blockIdx.x - row * splits;
  const int r = in.R - 1 - row;
  const int v0 = sp * seg;
  const int n = min(seg, in.V - v0);
  const int nv = n / X::N, left = n - nv * X::N;
  char* dx = dx_all + ((long long)r * in.V + v0) * X::size;
  float a = kp.coef[r];
  if (a != 0.f) {
    if (up.per == LM_UP_ALL)
      a *= up.g[0] * *kp.inv;
    else
      a *= up.g[up.per == LM_UP_ROW ? r : (r / in.T) % up.pairs];
  }
  if (a == 0.f) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int i = tid; i < nv; i += kThreads)
      *(u32x4_any*)(dx + (long long)i * 16) = zero;
    if (tid < left) X::put(dx + (long long)(nv * X::N + tid) * X::size, 0.f);
    return;
  }
  const char* x = (const char*)in.x + (row_start(in, r) + v0) * X::size;
  const LmStat st = kp.stat[r];
  const float c = in.c, mb = st.mb, w = a * st.w;
  const long long target = ONE ? place(pl, r) - v0 : -1;
  constexpr int Q = 4;
  for (int i = tid; i < nv; i += Q * kThreads) {
    u32x4 raw[Q];
#pragma unroll
    for (int g = 0; g < Q; ++g)
      if (i + g * kThreads < nv)
        raw[g] = *(const u32x4_any*)(x + (long long)(i + g * kThreads) * 16);
#pragma unroll
    for (int g = 0; g < Q; ++g) {
      const int ig = i + g * kThreads;
      if (ig >= nv) break;
      float f[X::N];
      X::open(raw[g], f);
#pragma unroll
      for (int e = 0; e < X::N; ++e) f[e] = w * exp2_hw((f[e] - mb) * c);
      if (ONE && target >= (long long)ig * X::N &&
          target < (long long)(ig + 1) * X::N) {
#pragma unroll
        for (int e = 0; e < X::N; ++e)
          if (target == (long long)ig * X::N + e) f[e] -= a;
      }
      *(u32x4_any*)(dx + (long long)ig * 16) = X::close(f);
    }
  }
  if (tid < left) {
    const int j = nv * X::N + tid;
    float f = w * exp2_hw((X::one(x + (long long)j * X::size) - mb) * c);
    if (ONE && target == j) f -= a;
    X::put(dx + (long long)j * X::size, f);
  }
  if (!ONE) {
    // the record's places: the same index twice adds both probabilities, and
    // both threads write the same value
    if (tid < pl.K) {
      s_idx[tid] = place(pl, (long long)r * pl.K + tid) - v0;
      s_p[tid] = kp.p[(long long)r * pl.K + tid];
    }
    __syncthreads();
    if (tid < pl.K) {
      const long long j = s_idx[tid];
      if (j >= 0 && j < n) {
        float ps = 0.f;
        for (int k = 0; k < pl.K; ++k) ps += s_idx[k] == j ? s_p[k] : 0.f;
        const float q =
            st.mass_S * exp2_hw((X::one(x + j * X::size) - st.M) * c);
        X::put(dx + j * X::size, a * (q - ps));
      }
    }
  }
}

// --------------------------------------------------------------------- topk
// One block per row. Thread c owns the vectors c, c + THREADS, ...; the k-th
// largest of the threads' maxima is a bound below the k-th largest logit, as
// k logits reach it. Only the threads' shares whose maximum reaches the bound
// are read again (about k of them, so some k/THREADS of the row, from the
// cache), and the few logits that reach it are ranked by counting. Rows that
// break this (a long run of equal logits, fewer finite ones than k) find the
// k-th key by bisection over the whole row.
DEVINL unsigned order_key(float f) {
  if (f != f) return 0xffffffffu;  // above all, as in torch
  unsigned u = __float_as_uint(f + 0.f);  // -0 and 0 are equal
  return u ^ ((int)u < 0 ? 0xffffffffu : 0x80000000u);
}

constexpr int kCand = 1024;

template <int TY, int THREADS>
__global__ void __launch_bounds__(THREADS)
    lm_topk_kernel(LmRows in, float temperature, int k, char* __restrict__ values,
                   long long* __restrict__ indices, float* __restrict__ lse) {
  using X = Ty<TY>;
  __shared__ Run red[THREADS / 64];
  __shared__ unsigned keys[THREADS];
  __shared__ unsigned long long cand[kCand];
  __shared__ int share[THREADS];
  __shared__ int n_share, n_cand, total;
  __shared__ unsigned s_bound;
  const int tid = threadIdx.x, r = blockIdx.x;
  const char* x = (const char*)in.x + row_start(in, r) * X::size;
  const float c = in.c;
  const int V = in.V, nv = V / X::N, left = V - nv * X::N;
  if (tid == 0) n_share = n_cand = 0;

  Run a = run_empty();
  float mx = -INFINITY;
  constexpr int Q = 4;
  for (int i = tid; i < nv; i += Q * THREADS) {
    float f[Q * X::N];
#pragma unroll
    for (int g = 0; g < Q; ++g) {
      const int ig = i + g * THREADS;
      if (ig < nv) {
        u32x4 raw = *(const u32x4_any*)(x + (long long)ig * 16);
        X::open(raw, f + g * X::N);
      } else {
#pragma unroll
        for (int e = 0; e < X::N; ++e) f[g * X::N + e] = -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < Q * X::N; ++e) mx = fmaxf(mx, f[e]);
    const float vm = fmaxf(a.m, mx);
    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < Q * X::N; ++e) add[e & 3] += exp_of(f[e] - vm, in);
    a.s = a.s * exp_of(a.m - vm, in) + ((add[0] + add[1]) + (add[2] + add[3]));
    a.m = vm;
  }
  // a NaN hides from fmaxf but not from the sum; +inf, which also makes the
  // sum one, is a bound below either
  unsigned key = tid < nv ? order_key(a.s != a.s ? INFINITY : mx) : 0u;
  keys[tid] = key;
  if (tid < left) a.join(X::one(x + (long long)(nv * X::N + tid) * X::size), 1.f, c);
  a = block_join<THREADS>(a, c, red);
  if (tid == 0)  // a row of -inf: log 0
    lse[r] = (float)((double)a.m / temperature + log((double)a.s));
  if (tid < 64) {
    unsigned mine[THREADS / 64], t = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) mine[i] = keys[i * 64 + tid];
    for (int bit = 31; bit >= X::low_bits; --bit) {
      const unsigned trial = t | (1u << bit);
      int cnt = 0;
#pragma unroll
      for (int i = 0; i < THREADS / 64; ++i)
        cnt += __popcll(__ballot(mine[i] >= trial));
      if (cnt >= k) {
        t = trial;
        if (cnt <= k + (k >> 2)) break;  // near enough
      }
    }
    if (tid == 0) s_bound = t;
  }
  __syncthreads();
  const unsigned bound = s_bound;
  auto offer = [&](float f, int j) {
    const unsigned o = order_key(f);
    if (o >= bound) {
      const int at = atomicAdd(&n_cand, 1);
      if (at < kCand)
        cand[at] = (unsigned long long)o << 32 | (0xffffffffu - (unsigned)j);
    }
  };
  if (key >= bound && tid < nv) share[atomicAdd(&n_share, 1)] = tid;
  if (tid < left) offer(X::one(x + (long long)(nv * X::N + tid) * X::size), nv * X::N + tid);
  __syncthreads();
  const int deep = (nv + THREADS - 1) / THREADS, work = n_share * deep;
  for (int i = tid; i < work; i += THREADS) {
    const int q = i / deep;
    const int ig = share[q] + (i - q * deep) * THREADS;
    if (ig < nv) {
      float f[X::N];
      X::open(*(const u32x4_any*)(x + (long long)ig * 16), f);
#pragma unroll
      for (int e = 0; e < X::N; ++e) offer(f[e], ig * X::N + e);
    }
  }
  __syncthreads();
  int nc = n_cand;
  if (nc > kCand || nc < k) {
    // the k-th largest (key, place) by bisection, all keys being different
    unsigned long long t = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long trial = t | 1ull << bit;
      __syncthreads();
      if (tid == 0) total = 0;
      __syncthreads();
      int mine = 0;
      for (int j = tid; j < V; j += THREADS) {
        const unsigned long long o =
            (unsigned long long)order_key(X::one(x + (long long)j * X::size)) << 32 |
            (0xffffffffu - (unsigned)j);
        mine += o >= trial;
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) mine += __shfl_xor(mine, off, 64);
      if ((tid & 63) == 0) atomicAdd(&total, mine);
      __syncthreads();
      if (total >= k) t = trial;
    }
    __syncthreads();
    if (tid == 0) n_cand = 0;
    __syncthreads();
    for (int j = tid; j < V; j += THREADS) {
      const unsigned long long o =
          (unsigned long long)order_key(X::one(x + (long long)j * X::size)) << 32 |
          (0xffffffffu - (unsigned)j);
      if (o >= t) cand[atomicAdd(&n_cand, 1)] = o;
    }
    __syncthreads();
    nc = n_cand;
  }
  for (int i = tid; i < nc; i += THREADS) {
    const unsigned long long mine = cand[i];
    int rank = 0;
    for (int q = 0; q < nc; ++q) rank += cand[q] > mine;
    if (rank < k) {
      const unsigned j = 0xffffffffu - (unsigned)mine;
      const long long at = (long long)r * k + rank;
      indices[at] = j;
      if (X::size == 2)
        ((short*)values)[at] = ((const short*)x)[j];
      else
        ((int*)values)[at] = ((const int*)x)[j];
    }
  }
}

int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// Splits of a row over blocks: enough blocks to fill the chip, none with less
// than one vector per thread.
int splits_for(const LmRows& in, int blocks, int seg_most, int* seg) {
  const int per = kThreads * (in.type == LM_FP32 ? 4 : 8);
  int s = div_up(blocks, in.R);
  s = std::min(s, std::max(1, div_up(in.V, per)));
  s = std::max(s, div_up(in.V, seg_most));
  // whole vectors per thread, so that segments start where vectors do
  *seg = div_up(div_up(in.V, s), 32) * 32;
  return div_up(in.V, *seg);
}

constexpr int kStatBlocks = 1024, kStatSeg = 131072;
constexpr int kGradBlocks = 2048, kGradSeg = 32768;

template <int TY>
void grad_of(const LmRows& in, const LmPlaces& pl, const LmKeep& kp,
             const LmUp& up, void* dx, hipStream_t s) {
  int seg;
  const int splits = splits_for(in, kGradBlocks, kGradSeg, &seg);
  const dim3 grid((unsigned)in.R * splits);
  if (!kp.p)
    lm_grad_kernel<TY, true><<<grid, kThreads, 0, s>>>(in, pl, kp, up,
                                                       (char*)dx, splits, seg);
  else
    lm_grad_kernel<TY, false><<<grid, kThreads, 0, s>>>(in, pl, kp, up,
                                                        (char*)dx, splits, seg);
}

template <int TY>
void stats_of(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
              const LmWork& w, const LmKeep& kp, hipStream_t s) {
  int seg;
  const int splits = splits_for(in, kStatBlocks, kStatSeg, &seg);
  const dim3 grid((unsigned)in.R * (splits + (te.values ? 1 : 0)));
  if (w.part_top)
    lm_stats_kernel<TY, true><<<grid, kThreads, (seg + 31) / 32 * 4, s>>>(
        in, pl, te, splits, seg, w.part, w.part_top, kp.p, w.rec, w.counter);
  else
    lm_stats_kernel<TY, false><<<grid, kThreads, 0, s>>>(
        in, pl, te, splits, seg, w.part, w.part_top, kp.p, w.rec, w.counter);
}

template <int TY>
void topk_of(const LmRows& in, float temperature, int k, void* values,
             long long* indices, float* lse, hipStream_t s) {
  lm_topk_kernel<TY, 1024><<<dim3(in.R), 1024, 0, s>>>(
      in, temperature, k, (char*)values, indices, lse);
}

#define LM_BY_TYPE(type, call)            \
  do {                                    \
    if ((type) == LM_BF16) {              \
      constexpr int TY = LM_BF16;         \
      call;                               \
    } else if ((type) == LM_FP16) {       \
      constexpr int TY = LM_FP16;         \
      call;                               \
    } else {                              \
      constexpr int TY = LM_FP32;         \
      call;                               \
    }                                     \
  } while (0)

void stats(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
           const LmWork& w, const LmKeep& kp, hipStream_t s) {
  LM_BY_TYPE(in.type, (stats_of<TY>(in, pl, te, w, kp, s)));
}

}  // namespace

int lm_stats_splits(const LmRows& in) {
  int seg;
  return splits_for(in, kStatBlocks, kStatSeg, &seg);
}

int lm_grad_splits(const LmRows& in) {
  int seg;
  return splits_for(in, kGradBlocks, kGradSeg, &seg);
}

int lm_blocks_of_rows(int R) { return div_up(R, kThreads); }

void lm_distill(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
                const LmWork& w, const LmKeep& kp, const LmOut& o,
                hipStream_t s) {
  stats(in, pl, te, w, kp, s);
  lm_distill_kernel<<<dim3(lm_blocks_of_rows(in.R)), kThreads, 0, s>>>(
      in, pl, te, w.splits, w.part, w.part_top, w.rec, kp.stat, kp.coef,
      w.bpart, w.counter, o);
}

void lm_policy(const LmRows& in, const LmPlaces& pl, const LmPolicy& po,
               const LmWork& w, const LmKeep& kp, float* logps, float* kl,
               const LmOut& o, hipStream_t s) {
  stats(in, pl, LmTeacher{}, w, kp, s);
  lm_policy_kernel<<<dim3(lm_blocks_of_rows(in.R)), kThreads, 0, s>>>(
      in, pl, po, w.splits, w.part, kp.stat, kp.coef, logps, kl, w.bpart,
      w.counter, o);
}

void lm_preference(const LmRows& in, const LmPlaces& pl, const LmPreference& pr,
                   const LmWork& w, const LmKeep& kp, float* chosen,
                   float* rejected, const LmOut& o, hipStream_t s) {
  stats(in, pl, LmTeacher{}, w, kp, s);
  const int pairs = in.R / in.T / 2;
  const int threads = std::min(1024, std::max(64, div_up(in.T, 64) * 64));
  lm_preference_kernel<<<dim3(pairs), threads, 0, s>>>(
      in, pl, pr, w.splits, w.part, kp.stat, kp.coef, chosen, rejected, w.bpart,
      w.counter, o);
}

void lm_grad(const LmRows& in, const LmPlaces& pl, const LmKeep& kp,
             const LmUp& up, void* dx, hipStream_t s) {
  LM_BY_TYPE(in.type, (grad_of<TY>(in, pl, kp, up, dx, s)));
}

void lm_topk(const LmRows& in, float temperature, int k, void* values,
             long long* indices, float* lse, hipStream_t s) {
  LM_BY_TYPE(in.type, (topk_of<TY>(in, temperature, k, values, indices, lse, s)));
}
