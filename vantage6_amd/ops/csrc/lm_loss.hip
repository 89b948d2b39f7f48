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
#include <type_traits>

namespace {

constexpr int kThreads = 256;
constexpr int Q = 4;  // 16-byte loads in flight per thread
constexpr double kLog2e = 1.4426950408889634074;

// 16 bytes at the alignment of one element: rows of an odd V start anywhere.
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
typedef float f32x8_v __attribute__((ext_vector_type(8)));

// With NT the load or store asks not to stay in the caches.
template <bool NT>
DEVINL u32x4 load16(const char* p) {
  if (NT) return __builtin_nontemporal_load((const u32x4_any*)p);
  return *(const u32x4_any*)p;
}
template <bool NT>
DEVINL void store16(char* p, u32x4 v) {
  if (NT)
    __builtin_nontemporal_store(v, (u32x4_any*)p);
  else
    *(u32x4_any*)p = v;
}

template <int TY>
struct Ty;
template <>
struct Ty<LM_BF16> {
  static constexpr int N = 8, size = 2, low_bits = 16;
  static DEVINL u32x4 lowest() { return u32x4(0xff80ff80u); }  // -inf
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
  static DEVINL u32x4 lowest() { return u32x4(0xfc00fc00u); }
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
  static DEVINL u32x4 lowest() { return u32x4(0xff800000u); }
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

// A stretch of n elements at p as vectors that begin where a cache line does,
// and up to 70 loose elements before and behind them. A wave's store of 1 KB
// then covers whole lines: the gradient of 4096 rows of 30522 fp16 logits, which
// begin anywhere in a line, took 68 us in vectors from each row's start and takes
// 56, that of rows of 30521 76 and 56.
struct Cut {
  int head, nv, loose;
};
template <int TY>
DEVINL Cut cut_of(const char* p, int n) {
  using X = Ty<TY>;
  const int to_line = (int)((128 - ((uintptr_t)p & 127)) & 127) / X::size;
  const int head = min(n, to_line), nv = (n - head) / X::N;
  return {head, nv, n - nv * X::N};
}
// where loose element i < loose lies, and where vector i begins
template <int TY>
DEVINL int loose_at(const Cut& cut, int i) {
  return i < cut.head ? i : i + cut.nv * Ty<TY>::N;
}

// 2^a by the hardware instruction: results under 2^-126 are 0, which changes
// no sum that has a term of 1 and no probability that a float can tell from 0.
DEVINL float exp2_hw(float a) { return __builtin_amdgcn_exp2f(a); }

// 2^(d log2(e)/t) with the constant in two parts: one float of it is off by up
// to 2^-25, the same way for every logit, and that would be 1e-7 in log S, in
// one direction for all the tokens of an answer. Both parts are positive, so
// that a d of -inf stays one.
DEVINL float exp_of(float d, const LmRows& in) {
  return exp2_hw(fmaf(d, in.c_hi, d * in.c_lo));
}

// Reductions over a wave by DPP moves, a few cycles each where a shuffle
// through LDS takes a hundred: lane ^ 1, lane ^ 2, 7 - lane of 8, 15 - lane of
// 16, then the four rows' results. Every lane of the wave has to be there.
template <int CTRL>
DEVINL float moved(float v) {
  return __int_as_float(
      __builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 15, 15, true));
}
DEVINL float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
DEVINL float max_of_8(float v) {
  v = fmaxf(v, moved<0xB1>(v));
  v = fmaxf(v, moved<0x4E>(v));
  return fmaxf(v, moved<0x141>(v));
}
DEVINL float wave_max(float v) {
  v = max_of_8(v);
  v = fmaxf(v, moved<0x140>(v));
  return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)),
               fmaxf(lane_of(v, 32), lane_of(v, 48)));
}
DEVINL float wave_add(float v) {
  v += moved<0xB1>(v);
  v += moved<0x4E>(v);
  v += moved<0x141>(v);
  v += moved<0x140>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// A running maximum and the sum of 2^((x-m)c) below it. m starts at the least
// finite float, so that -inf adds 0 and never meets itself in a difference.
struct Run {
  float m, s;
  DEVINL void join(float om, float os, const LmRows& in) {
    const float mn = fmaxf(m, om);
    s = s * exp_of(m - mn, in) + os * exp_of(om - mn, in);
    m = mn;
  }
};
DEVINL Run run_empty() { return {-FLT_MAX, 0.f}; }
DEVINL Run wave_join(Run a, const LmRows& in) {
  const float m = wave_max(a.m);
  return {m, wave_add(a.s * exp_of(a.m - m, in))};
}

template <int THREADS>
DEVINL Run block_join(Run a, const LmRows& in, Run* red) {
  a = wave_join(a, in);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) a.join(red[w].m, red[w].s, in);
  return a;
}

DEVINL double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// two sums over a block in every thread, in one order
DEVINL void block_sum2(double& a, double& b, double2* red) {
  a = wave_sum(a);
  b = wave_sum(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_double2(a, b);
  __syncthreads();
  a = b = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
    a += red[w].x;
    b += red[w].y;
  }
}

// A record's probabilities by one wave, up to 4 of its 256 entries a lane, in
// 64 bits as 1 - sum p follows. rec = {sum p log p, sum p (x - x_ref), sum p,
// x_ref}, sum p < 0 marks a row without a record. x_ref is the largest of the
// record's logits: sums of p x and of p M would cancel where all of them are the
// type's lowest value, and leave 1e22 of 1e38.
DEVINL void record_of(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
                      int r, float* p_out, double4* rec) {
  constexpr int E = kLmMostK / 64;
  const int lane = threadIdx.x & 63;
  const long long at = (long long)r * pl.K, x_at = row_start(in, r);
  const double t = te.temperature;
  long long j[E];
  float v[E], m = -INFINITY;
  bool any = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int k = lane + 64 * e;
    j[e] = k < pl.K ? place(pl, at + k) : -1;
    v[e] = j[e] >= 0 ? one_of(te.type, (const char*)te.values, at + k) : -INFINITY;
    any |= !(v[e] == -INFINITY);
    m = fmaxf(m, v[e]);
  }
  if (!__any(any)) {
    if (lane == 0) rec[r] = make_double4(0, 0, -1, 0);
    return;
  }
  double lp[E], z = 0.0;
  if (te.lse) {
#pragma unroll
    for (int e = 0; e < E; ++e) lp[e] = (double)v[e] / t - te.lse[r];
  } else {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (64 * e >= pl.K) break;
      lp[e] = ((double)v[e] - m) / t;
      z += v[e] == -INFINITY ? 0.0 : exp(lp[e]);
    }
    z = log(wave_sum(z));
  }
  double a = 0.0, b = 0.0, sum = 0.0, x_ref = -FLT_MAX;  // the lane's, so far
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (64 * e >= pl.K) break;
    if (!te.lse) lp[e] -= z;
    double p = v[e] == -INFINITY ? 0.0 : exp(lp[e]);
    // a place outside the row makes it a NaN, though its p may be 0
    if (j[e] >= in.V && v[e] != -INFINITY) p = NAN;
    if (p != 0.0) {
      const double x = j[e] < in.V
          ? (double)one_of(in.type, (const char*)in.x, x_at + j[e]) : NAN;
      a += p * lp[e];
      if (x > x_ref) {
        b += sum * (x_ref - x);
        x_ref = x;
      }
      b += p * (x - x_ref);
      sum += p;
    }
    if (lane + 64 * e < pl.K) p_out[at + lane + 64 * e] = (float)p;
  }
  const double x_all = wave_max((float)x_ref);
  b += sum * (x_ref - x_all);
  a = wave_sum(a);
  b = wave_sum(b);
  sum = wave_sum(sum);
  if (lane == 0) rec[r] = make_double4(a, b, sum, x_all);
}

// ------------------------------------------------------------------- stats
// Per row `splits` blocks, block s of which takes `seg` logits from s*seg on;
// before them the blocks that make a distillation's records, a row per wave
// (after them they would be a tail). With TOP, the K places of a record are
// kept apart: a bit per logit of the segment in LDS, so that the sum outside
// the record is one of its own and not the difference of two that nearly
// cancel.
template <int TY, int THREADS, bool REC, bool TOP>
__global__ void __launch_bounds__(THREADS)
    lm_stats_kernel(LmRows in, LmPlaces pl, LmTeacher te, int splits, int seg,
                    int keep16, float2* __restrict__ part,
                    float2* __restrict__ part_top, float* __restrict__ xt,
                    float* __restrict__ p, double4* __restrict__ rec,
                    int* __restrict__ counter) {
  using X = Ty<TY>;
  extern __shared__ unsigned bits[];
  __shared__ Run red[THREADS / 64];
  const int tid = threadIdx.x;
  if (blockIdx.x == 0 && tid == 0) *counter = 0;  // for the finish kernel
  int block = blockIdx.x;
  if (REC) {
    constexpr int W = THREADS / 64;
    const int records = (in.R + W - 1) / W;
    if (block < records) {
      const int r = block * W + (tid >> 6);
      if (r < in.R && !ignored(pl, r)) record_of(in, pl, te, r, p, rec);
      return;
    }
    block -= records;
  }
  const int r = block / splits, sp = block - r * splits;
  if (ignored(pl, r)) return;
  const int v0 = sp * seg;
  const int n = min(seg, in.V - v0);
  const char* x = (const char*)in.x + (row_start(in, r) + v0) * X::size;
  const Cut cut = cut_of<TY>(x, n);
  const int nv = cut.nv;
  const char* xv = x + cut.head * X::size;
  const bool stay = (r & 15) < keep16;
  u32x4 first[Q];
#pragma unroll
  for (int g = 0; g < Q; ++g) first[g] = X::lowest();
  // two loops of loads, kept apart: the compiler would join equal loads of
  // both branches and drop the hint
  if (stay) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int g = 0; g < Q; ++g)
      if (tid + g * THREADS < nv)
        first[g] = load16<false>(xv + (long long)(tid + g * THREADS) * 16);
  } else {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int g = 0; g < Q; ++g)
      if (tid + g * THREADS < nv)
        first[g] = load16<true>(xv + (long long)(tid + g * THREADS) * 16);
  }
  if (xt && tid == 0) {
    const long long j = place(pl, r);
    if (j >= v0 && j < v0 + n)
      xt[r] = X::one(x + (j - v0) * X::size);
    else if (sp == 0 && (j < 0 || j >= in.V))
      xt[r] = NAN;  // a place outside the row
  }
  const int loose_bits = (nv * X::N + 31) / 32 * 32;
  if (TOP) {
    // the vectors' elements from 0 on, the loose ones behind them
    for (int i = tid; i < loose_bits / 32 + 3; i += THREADS) bits[i] = 0;
    __syncthreads();
    for (int k = tid; k < pl.K; k += THREADS) {
      const long long at = place(pl, (long long)r * pl.K + k) - v0;
      if (at >= 0 && at < n) {
        const int j = (int)at;
        const int b = j < cut.head                  ? loose_bits + j
                      : j >= cut.head + nv * X::N ? loose_bits + j - nv * X::N
                                                  : j - cut.head;
        atomicOr(&bits[b >> 5], 1u << (b & 31));
      }
    }
    __syncthreads();
  }
  Run a = run_empty(), top = run_empty();
  auto take = [&](const u32x4* raw, int i) {
    float f[Q * X::N];
#pragma unroll
    for (int g = 0; g < Q; ++g) X::open(raw[g], f + g * X::N);
    if (TOP) {
#pragma unroll
      for (int g = 0; g < Q; ++g) {
        const int j = (i + g * THREADS) * X::N;
        unsigned hit = j < nv * X::N ? bits[j >> 5] >> (j & 31) : 0u;
        hit &= (1u << X::N) - 1u;
        if (hit) {
#pragma unroll
          for (int e = 0; e < X::N; ++e)
            if (hit >> e & 1) {
              top.join(f[g * X::N + e], 1.f, in);
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
  };
  take(first, tid);
  auto walk = [&](auto nt) {
    int i = tid + Q * THREADS;
    for (; i + (Q - 1) * THREADS < nv; i += Q * THREADS) {
      u32x4 raw[Q];
#pragma unroll
      for (int g = 0; g < Q; ++g)
        raw[g] = load16<nt.value>(xv + (long long)(i + g * THREADS) * 16);
      take(raw, i);
    }
    if (i < nv) {
      u32x4 raw[Q];
#pragma unroll
      for (int g = 0; g < Q; ++g) {
        raw[g] = X::lowest();
        if (i + g * THREADS < nv)
          raw[g] = load16<nt.value>(xv + (long long)(i + g * THREADS) * 16);
      }
      take(raw, i);
    }
  };
  if (stay)
    walk(std::false_type());
  else
    walk(std::true_type());
  for (int i = tid; i < cut.loose; i += THREADS) {
    const float f = X::one(x + loose_at<TY>(cut, i) * X::size);
    const int b = loose_bits + i;
    if (TOP && (bits[b >> 5] >> (b & 31) & 1))
      top.join(f, 1.f, in);
    else
      a.join(f, 1.f, in);
  }
  a = block_join<THREADS>(a, in, red);
  if (TOP) {
    __syncthreads();
    top = block_join<THREADS>(top, in, red);
  }
  if (tid == 0) {
    const long long at = (long long)r * splits + sp;
    part[at] = make_float2(a.m, a.s);
    if (TOP) part_top[at] = make_float2(top.m, top.s);
  }
}

// The finish kernels give a row to a group of lanes, a power of two that holds
// the row's splits (at most a wave), and work in 64 bits from here on.
struct Row {
  double m, s;
};
DEVINL Row join_splits(const float2* part, int splits, int group, int r,
                       bool live, double c) {
  const int lane = threadIdx.x & (group - 1);
  float m = -FLT_MAX;
  double s = 0.0;
  if (live)
    for (int i = lane; i < splits; i += group) {
      const float2 q = part[(long long)r * splits + i];
      const float mn = fmaxf(m, q.x);
      if (m != mn) s *= exp2(((double)m - mn) * c);
      s += q.x == mn ? (double)q.y : (double)q.y * exp2(((double)q.x - mn) * c);
      m = mn;
    }
  float all = m;
  for (int off = 1; off < group; off <<= 1)
    all = fmaxf(all, __shfl_xor(all, off, 64));
  if (m != all) s *= exp2(((double)m - all) * c);
  for (int off = 1; off < group; off <<= 1) s += __shfl_xor(s, off, 64);
  m = all;
  return {(double)m, s};
}

// Sum over the whole grid of a block's `loss` and `count`, as its first thread
// has them, in one order: each block's sums in memory, the block that arrives
// last adds them up. *o.loss = the loss, *o.inv = 1/count for a mean over what
// counts, else 1.
DEVINL void grid_mean(double loss, double count, double2* bpart, int* counter,
                      const LmOut& o) {
  __shared__ double2 red[16];
  __shared__ int last;
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
    block_sum2(loss, count, red);
  }
  if (threadIdx.x == 0) {
    const double inv = o.reduction == LM_MEAN ? 1.0 / fmax(count, 1.0) : 1.0;
    *o.loss = (float)(loss * inv);
    *o.inv = (float)inv;
  }
}

// The same of a row's loss per lane that leads one.
DEVINL void grid_mean_of_rows(double loss, bool lead, bool live, const LmWork& w,
                              const LmOut& o) {
  __shared__ double2 red[16];
  if (o.reduction == LM_NONE) return;
  double count = lead && live ? 1.0 : 0.0;
  loss = lead ? loss : 0.0;
  block_sum2(loss, count, red);
  grid_mean(loss, count, w.bpart, w.counter, o);
}

// ------------------------------------------------------------------ distill
__global__ void __launch_bounds__(kThreads)
    lm_distill_kernel(LmRows in, LmPlaces pl, LmTeacher te, LmWork w, LmKeep kp,
                      LmOut o) {
  const int at = blockIdx.x * blockDim.x + threadIdx.x, r = at / w.group;
  const bool lead = (at & (w.group - 1)) == 0 && r < in.R;
  const bool on = r < in.R && !ignored(pl, r);
  const double4 k = on ? w.rec[r] : make_double4(0, 0, -1, 0);
  const bool live = !(k.z < 0.0);
  const double t = te.temperature, c = kLog2e / t;
  const Row rest = join_splits(w.part, w.splits, w.group, r, live, c);
  Row top = {0, 0};
  if (te.lse) top = join_splits(w.part_top, w.splits, w.group, r, live, c);
  LmStat st = {0.f, 0.f, 0.f, 0.f};
  double loss = 0.0;
  float a = 0.f;
  if (live) {
    Row all = rest;
    // dL/dx_j t = mass q_j - p_j, mass = sum p + rest: 1, if the record's
    // values and its logsumexp are of the same row
    double tail = 0.0, mass = k.z;
    if (te.lse) {
      const double p_rest = fmax(1.0 - k.z, 0.0);
      all.m = fmax(rest.m, top.m);
      all.s = rest.s * exp((rest.m - all.m) / t) + top.s * exp((top.m - all.m) / t);
      // no logit outside the record is above -inf: it has no rest
      if (rest.s != 0.0) {
        const double log_rest = (rest.m - all.m) / t + log(rest.s / all.s);
        if (p_rest > 0.0) tail = p_rest * (log(p_rest) - log_rest);
        mass += p_rest;
        st.w = (float)((mass * exp(log_rest) - p_rest) / rest.s);
      }
    } else {
      st.w = (float)(mass / all.s);
    }
    st.mb = (float)rest.m;
    st.M = (float)all.m;
    st.mass_S = (float)(mass / all.s);
    // sum p (log p - log q)
    loss = t * t * (k.x - (k.y + k.z * (k.w - all.m)) / t + k.z * log(all.s) + tail);
    // d/dx of t^2 KL(x/t); a NaN, of a place outside the row too, is the
    // whole row's
    a = loss == loss ? (float)t : NAN;
  }
  if (lead) {
    kp.stat[r] = st;
    kp.coef[r] = a;
    if (o.reduction == LM_NONE) o.loss[r] = (float)loss;
  }
  grid_mean_of_rows(loss, lead, live, w, o);
}

// ------------------------------------------- log-probability of one token
// lp = (x_t - M) - log S; a target outside the row gives NaN
DEVINL double token_logp(const LmWork& w, int r, bool live, LmStat* st) {
  const Row a = join_splits(w.part, w.splits, w.group, r, live, kLog2e);
  *st = {0.f, 0.f, 0.f, 0.f};
  if (!live) return 0.0;
  const float inv = (float)(1.0 / a.s);
  *st = {(float)a.m, inv, (float)a.m, inv};
  return ((double)w.xt[r] - a.m) - log(a.s);
}

__global__ void __launch_bounds__(kThreads)
    lm_policy_kernel(LmRows in, LmPlaces pl, LmPolicy po, LmWork w, LmKeep kp,
                     float* __restrict__ logps, float* __restrict__ kls,
                     LmOut o) {
  const int at = blockIdx.x * blockDim.x + threadIdx.x, r = at / w.group;
  const bool lead = (at & (w.group - 1)) == 0 && r < in.R;
  const bool live = r < in.R && !ignored(pl, r);
  double loss = 0.0, by_lp = 0.0, kl = 0.0;
  LmStat st;
  const double lp = token_logp(w, r, live, &st);
  if (live) {
    const double A = po.adv[r], lo = 1.0 - po.clip_low, hi = 1.0 + po.clip_high;
    const double ratio = exp(lp - (double)po.old_lp[r]);
    const double held = fmin(fmax(ratio, lo), hi);
    // the lesser of ratio*A and held*A; a NaN stays one
    const bool moves = A > 0.0 ? !(ratio > hi) : !(ratio < lo) || A != A;
    loss = moves ? -ratio * A : -held * A;
    by_lp = moves ? -ratio * A : 0.0;
    if (po.ref_lp) {
      const double d = (double)po.ref_lp[r] - lp, e = expm1(d);
      kl = e - d;
      // without weight it is reported only: it may be +inf, and 0 * inf a NaN
      if (po.kl_coef != 0.0) {
        loss += po.kl_coef * kl;
        by_lp -= po.kl_coef * e;
      }
    }
  }
  if (lead) {
    kp.stat[r] = st;
    kp.coef[r] = (float)-by_lp;  // the gradient is coef * (q - onehot)
    logps[r] = (float)lp;
    kls[r] = (float)kl;
    if (o.reduction == LM_NONE) o.loss[r] = (float)loss;
  }
  grid_mean_of_rows(loss, lead, live, w, o);
}

// One block per pair: sequences n and n + N. The sums over an answer are held
// in 64 bits, as the loss is made of the small differences between them.
__global__ void __launch_bounds__(1024)
    lm_preference_kernel(LmRows in, LmPlaces pl, LmPreference pr, LmWork w,
                         LmKeep kp, float* __restrict__ chosen,
                         float* __restrict__ rejected, LmOut o) {
  __shared__ double2 red[16];
  __shared__ float s_a;
  const int n = blockIdx.x, N = gridDim.x, T = in.T;
  const int mine = threadIdx.x / w.group, rows = blockDim.x / w.group;
  const bool lead = (threadIdx.x & (w.group - 1)) == 0;
  double sum[2] = {0.0, 0.0};
  for (int t0 = 0; t0 < 2 * T; t0 += rows) {
    const int t = t0 + mine, side = t >= T;
    const int r = (n + side * N) * T + t - side * T;
    const bool live = t < 2 * T && !ignored(pl, r);
    LmStat st;
    const double lp = token_logp(w, r, live, &st);
    if (lead && t < 2 * T) {
      kp.stat[r] = st;
      sum[0] += side ? 0.0 : lp;
      sum[1] += side ? lp : 0.0;
    }
  }
  block_sum2(sum[0], sum[1], red);
  double loss = 0.0, z = 0.0, low = 0.0;
  if (threadIdx.x == 0) {
    double reward[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int b = n + side * N;
      const double ref = pr.ref64 ? ((const double*)pr.ref)[b]
                                  : (double)((const float*)pr.ref)[b];
      reward[side] = pr.beta * (sum[side] - ref);
    }
    z = reward[0] - reward[1];
    low = exp(-fabs(z));
    // 1 - sigmoid(z), without the difference
    const double away = (z < 0.0 ? 1.0 : low) / (1.0 + low);
    s_a = (float)(pr.beta * (away - pr.smoothing));
    chosen[n] = (float)reward[0];
    rejected[n] = (float)reward[1];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    // -log sigmoid(z) = max(-z, 0) + log(1 + exp(-|z|))
    const double e = pr.smoothing, both = log1p(low);
    loss = (1.0 - e) * (fmax(-z, 0.0) + both);
    if (e != 0.0) loss += e * (fmax(z, 0.0) + both);
    if (o.reduction == LM_NONE) o.loss[n] = (float)loss;
  }
  // the gradient is coef * (q - onehot), and the other way for the rejected
  const float a = s_a;
  for (int t = threadIdx.x; t < 2 * T; t += blockDim.x) {
    const int side = t >= T, r = (n + side * N) * T + t - side * T;
    kp.coef[r] = ignored(pl, r) ? 0.f : side ? -a : a;
  }
  if (o.reduction != LM_NONE) grid_mean(loss, 1.0, w.bpart, w.counter, o);
}

// --------------------------------------------------------------------- grad
// grid R*splits; block (r, s) reads its segment and writes the gradient. A row
// whose coefficient is 0 (ignored, or clipped) is not read. The rows go from
// the last to the first, as the last ones that stats read are the likeliest
// to be still in the cache.
template <int TY, bool ONE, bool NT>
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
  char* dx = dx_all + ((long long)r * in.V + v0) * X::size;
  const Cut cut = cut_of<TY>(dx, n);
  const int nv = cut.nv;
  char* dxv = dx + cut.head * X::size;
  float a = kp.coef[r];
  long long at = -1;  // the thread's place of the record
  float p = 0.f;
  if (!ONE && tid < pl.K) {
    at = place(pl, (long long)r * pl.K + tid) - v0;
    p = kp.p[(long long)r * pl.K + tid];
  }
  if (a != 0.f) {
    if (up.per == LM_UP_ALL)
      a *= up.g[0] * *kp.inv;
    else
      a *= up.g[up.per == LM_UP_ROW ? r : (r / in.T) % up.pairs];
  }
  if (a == 0.f) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int i = tid; i < nv; i += kThreads)
      store16<NT>(dxv + (long long)i * 16, zero);
    if (tid < cut.loose) X::put(dx + loose_at<TY>(cut, tid) * X::size, 0.f);
    return;
  }
  const char* x = (const char*)in.x + (row_start(in, r) + v0) * X::size;
  const char* xv = x + cut.head * X::size;
  const LmStat st = kp.stat[r];
  const float c = in.c, mb = st.mb, w = a * st.w;
  const long long target = ONE ? place(pl, r) - v0 : -1;
  // what goes to a place in this segment. The same index twice adds both
  // probabilities, and both threads write one value.
  float there = 0.f;
  if (!ONE) {
    if (tid < pl.K) {
      s_idx[tid] = at;
      s_p[tid] = p;
      if (at >= n) at = -1;
    }
    __syncthreads();
    if (at >= 0) {
      const float xt = X::one(x + at * X::size);
      float ps = 0.f;
      for (int k = 0; k < pl.K; ++k) ps += s_idx[k] == at ? s_p[k] : 0.f;
      there = a * (st.mass_S * exp2_hw((xt - st.M) * c) - ps);
    }
  }
  const long long aim = target - cut.head;
  auto put = [&](u32x4 raw, int ig) {
    float f[X::N];
    X::open(raw, f);
#pragma unroll
    for (int e = 0; e < X::N; ++e) f[e] = w * exp2_hw((f[e] - mb) * c);
    if (ONE && aim >= (long long)ig * X::N && aim < (long long)(ig + 1) * X::N) {
#pragma unroll
      for (int e = 0; e < X::N; ++e)
        if (aim == (long long)ig * X::N + e) f[e] -= a;
    }
    store16<NT>(dxv + (long long)ig * 16, X::close(f));
  };
  // rounds that a whole wave has, then what is left in one more (60000 rows of
  // 5001 bf16: vector by vector 208 us, so 176; with a record 220 and 200)
  int i = tid;
  for (; (i | 63) + (Q - 1) * kThreads < nv; i += Q * kThreads) {
    u32x4 raw[Q];
#pragma unroll
    for (int g = 0; g < Q; ++g)
      raw[g] = load16<true>(xv + (long long)(i + g * kThreads) * 16);
#pragma unroll
    for (int g = 0; g < Q; ++g) put(raw[g], i + g * kThreads);
  }
  if (i < nv) {
    u32x4 raw[Q];
#pragma unroll
    for (int g = 0; g < Q; ++g)
      if (i + g * kThreads < nv)
        raw[g] = load16<true>(xv + (long long)(i + g * kThreads) * 16);
#pragma unroll
    for (int g = 0; g < Q; ++g)
      if (i + g * kThreads < nv) put(raw[g], i + g * kThreads);
  }
  if (tid < cut.loose) {
    const int j = loose_at<TY>(cut, tid);
    float f = w * exp2_hw((X::one(x + j * X::size) - mb) * c);
    if (ONE && target == j) f -= a;
    X::put(dx + j * X::size, f);
  }
  if (!ONE) {
    __syncthreads();  // the row is written, now its places
    if (at >= 0) X::put(dx + at * X::size, there);
  }
}

// --------------------------------------------------------------------- topk
// One block per row. The row falls into pieces, and the k-th largest of their
// maxima is a bound below the k-th largest logit, as k logits reach it. Only
// the pieces whose maximum reaches the bound are read again, and the few logits
// that reach it are ranked by counting. A piece is one logit (PIECE = 0) where
// all fit into LDS, else a vector of 16 bytes, or a line of eight vectors where
// those are many: of 128256 logits in 16 bits 2004 lines, of which some k are
// read again. Rows that break this (a long run of equal logits, a NaN or +inf)
// find the k-th key by bisection over the whole row.
enum { kLogits = 0, kVectors = 1, kLines = 8 };

DEVINL unsigned order_of(float f) {  // not for a NaN
  const unsigned u = __float_as_uint(f + 0.f);  // -0 and 0 are equal
  return u ^ ((int)u < 0 ? 0xffffffffu : 0x80000000u);
}
DEVINL unsigned order_key(float f) {
  return f != f ? 0xffffffffu : order_of(f);  // above all, as in torch
}

constexpr int kCand = 1984;    // logits that reach the bound; four blocks fit a CU
constexpr int kPieces = 4096;  // maxima kept; piece i of a longer row is in i % kPieces

// a logit that ranks, its place, and whether its zero was a negative one
DEVINL unsigned long long candidate(float f, int j) {
  return (unsigned long long)order_key(f) << 32 | (unsigned)(0x3fffffff - j) << 1 |
         (__float_as_uint(f) == 0x80000000u);
}
DEVINL int place_of(unsigned long long cand) {
  return 0x3fffffff - (int)((unsigned)cand >> 1);
}
DEVINL float logit_of(unsigned long long cand) {
  const unsigned u = (unsigned)(cand >> 32);
  if (cand & 1) return -0.f;
  return __uint_as_float(u == 0xffffffffu ? 0x7fc00000u
                         : u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <int TY, int THREADS, int PIECE, bool NT>
__global__ void __launch_bounds__(THREADS)
    lm_topk_kernel(LmRows in, double temperature, int k,
                   char* __restrict__ values,
                   long long* __restrict__ indices, float* __restrict__ lse) {
  using X = Ty<TY>;
  __shared__ Run red[THREADS / 64];
  __shared__ __align__(16) float maxima[kPieces];
  __shared__ unsigned long long cand[kCand];
  __shared__ unsigned short share[kPieces];
  __shared__ int n_share, n_cand, total, odd;
  __shared__ float s_bound;
  __shared__ Run s_run;
  const int tid = threadIdx.x, r = blockIdx.x;
  const char* x = (const char*)in.x + row_start(in, r) * X::size;
  const float c = in.c;
  const int V = in.V;
  const Cut cut = cut_of<TY>(x, V);
  const int nv = cut.nv;
  const char* xv = x + cut.head * X::size;
  if (tid == 0) n_share = n_cand = odd = 0;
  for (int i = tid; i < kPieces; i += THREADS) maxima[i] = -INFINITY;
  __syncthreads();

  Run a = run_empty();
  constexpr int SHIFT = PIECE == kLines ? 3 : 0;  // vectors of a piece
  const int pieces = PIECE == kLogits ? V : (nv + (1 << SHIFT) - 1) >> SHIFT;
  const bool folded = pieces > kPieces;
  auto take = [&](const u32x4* raw, int i) {
    float f[Q * X::N], vm = a.m;
#pragma unroll
    for (int g = 0; g < Q; ++g) {
      X::open(raw[g], f + g * X::N);
      float m = f[g * X::N];
#pragma unroll
      for (int e = 1; e < X::N; ++e) m = fmaxf(m, f[g * X::N + e]);
      vm = fmaxf(vm, m);
      // one lane writes a place of `maxima`, in all rounds of a long row
      static_assert(kPieces % THREADS == 0, "a place has one writer");
      const int ig = i + g * THREADS;
      if (PIECE == kLogits) {
        if (ig < nv) {
#pragma unroll
          for (int e = 0; e < X::N; ++e) maxima[cut.head + ig * X::N + e] = f[g * X::N + e];
        }
        continue;
      }
      if (SHIFT) m = max_of_8(m);
      if ((!SHIFT || (tid & 7) == 0) && ig < nv) {
        float* at = &maxima[(ig >> SHIFT) & (kPieces - 1)];
        *at = folded ? fmaxf(*at, m) : m;
      }
    }
    // log S needs no second part of the constant here: 1e-7 is less than half
    // a step of its float
    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < Q * X::N; ++e) add[e & 3] += exp2_hw((f[e] - vm) * c);
    a.s = a.s * exp2_hw((a.m - vm) * c) + ((add[0] + add[1]) + (add[2] + add[3]));
    a.m = vm;
  };
  // whole waves go the same way: max_of_8 needs all its lanes
  int i = tid;
  for (; (i | 63) + (Q - 1) * THREADS < nv; i += Q * THREADS) {
    u32x4 raw[Q];
#pragma unroll
    for (int g = 0; g < Q; ++g)
      raw[g] = load16<NT>(xv + (long long)(i + g * THREADS) * 16);
    take(raw, i);
  }
  if ((i & ~63) < nv) {
    u32x4 raw[Q];
#pragma unroll
    for (int g = 0; g < Q; ++g) {
      raw[g] = X::lowest();
      if (i + g * THREADS < nv)
        raw[g] = load16<NT>(xv + (long long)(i + g * THREADS) * 16);
    }
    take(raw, i);
  }
  if (tid < cut.loose) {
    const int j = loose_at<TY>(cut, tid);
    const float f = X::one(x + j * X::size);
    if (PIECE == kLogits) maxima[j] = f;
    a.join(f, 1.f, in);
  }
  a = wave_join(a, in);
  if ((tid & 63) == 0) red[tid >> 6] = a;
  __syncthreads();
  if (tid < 64) {
    // The bound: any t that not many more than k maxima reach will do, and a few
    // maxima may go as one, which is a bound as well: 512 groups of them, or
    // 1024 where k is more than a quarter of that, as a bound that most groups
    // reach is a low one. Bit by bit from the first in which the finite ones
    // differ.
    constexpr int E = 16;
    const int groups = k <= 128 ? 512 : 1024;
    const int rounds = (min(pieces, kPieces) + groups - 1) / groups;
    unsigned mine[E];
    float m[E], least = INFINITY, most = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) m[e] = -INFINITY;
    for (int i = 0; i < rounds; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * 64 < groups) m[e] = fmaxf(m[e], maxima[i * groups + e * 64 + tid]);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      mine[e] = order_of(m[e]);
      least = fminf(least, m[e] > -INFINITY ? m[e] : INFINITY);
      most = fmaxf(most, m[e]);
    }
    const unsigned low = order_of(-wave_max(-least)), high = order_of(wave_max(most));
    auto reach = [&](unsigned trial) {
      int cnt = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e * 64 >= groups) break;
        cnt += __popcll(__builtin_amdgcn_ballot_w64(mine[e] >= trial));
      }
      return cnt;
    };
    unsigned t = 0;
    if (low <= high && reach(low) >= k) {  // else there are too few
      int bit = low == high ? -1 : 31 - __clz((int)(low ^ high));
      t = bit < 0 ? low : low & ~((2u << bit) - 1u);
      for (; bit >= X::low_bits; --bit) {
        const unsigned trial = t | (1u << bit);
        const int cnt = reach(trial);
        if (cnt >= k) {
          t = trial;
          if (cnt <= k + (k >> 3) + 4) break;
        }
      }
    }
    // keys up to that of -inf stand for no float
    if (tid == 0)
      s_bound = t <= order_of(-INFINITY) ? -INFINITY
                                          : logit_of((unsigned long long)t << 32);
  } else if (tid < 128) {
    // meanwhile another wave joins the sums
    constexpr int W = THREADS / 64;
    a = (tid & 63) < W ? red[tid & 63] : run_empty();
    a = wave_join(a, in);
    if (tid == 64) {
      s_run = a;
      // a NaN hides from fmaxf, but not from the sum, nor does a +inf, whose
      // difference from itself is one
      odd = a.s != a.s;
    }
  }
  __syncthreads();
  const float bound = s_bound;
  auto offer = [&](float f, int j) {
    const int at = atomicAdd(&n_cand, 1);
    if (at < kCand) cand[at] = candidate(f, j);
  };
  for (int i = tid; i < min(pieces, kPieces); i += THREADS)
    if (maxima[i] >= bound) {
      if (PIECE == kLogits)
        offer(maxima[i], i);
      else
        share[atomicAdd(&n_share, 1)] = (unsigned short)i;
    }
  if (PIECE != kLogits && tid < cut.loose) {
    const int j = loose_at<TY>(cut, tid);
    const float f = X::one(x + j * X::size);
    if (f >= bound) offer(f, j);
  }
  __syncthreads();
  if (PIECE != kLogits && !odd)
    for (int from = 0; from < pieces; from += kPieces) {
      const int work = n_share << SHIFT;
      for (int i = tid; i < work; i += THREADS) {
        const int ig = ((from + share[i >> SHIFT]) << SHIFT) + (i & ((1 << SHIFT) - 1));
        if (ig >= nv) continue;
        float f[X::N];
        X::open(load16<false>(xv + (long long)ig * 16), f);
        int hits = 0;
#pragma unroll
        for (int e = 0; e < X::N; ++e) hits += f[e] >= bound;
        if (!hits) continue;
        int at = atomicAdd(&n_cand, hits);
#pragma unroll
        for (int e = 0; e < X::N; ++e)
          if (f[e] >= bound) {
            if (at < kCand) cand[at] = candidate(f[e], cut.head + ig * X::N + e);
            ++at;
          }
      }
    }
  __syncthreads();
  int nc = n_cand;
  if (odd || nc > kCand || nc < k) {
    // The k-th largest (key, place) by bisection, all of them being different:
    // the bits of the key, then those of a place below V.
    auto each = [&](auto&& use) {
      for (int i = tid; i < nv; i += THREADS) {
        float f[X::N];
        X::open(load16<false>(xv + (long long)i * 16), f);
#pragma unroll
        for (int e = 0; e < X::N; ++e) use(candidate(f[e], cut.head + i * X::N + e));
      }
      if (tid < cut.loose) {
        const int j = loose_at<TY>(cut, tid);
        use(candidate(X::one(x + j * X::size), j));
      }
    };
    unsigned long long t = 0;
    auto settle = [&](int bit) {
      const unsigned long long trial = t | 1ull << bit;
      __syncthreads();
      if (tid == 0) total = 0;
      __syncthreads();
      int mine = 0;
      each([&](unsigned long long o) { mine += o >= trial; });
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) mine += __shfl_xor(mine, off, 64);
      if ((tid & 63) == 0) atomicAdd(&total, mine);
      __syncthreads();
      if (total >= k) t = trial;
    };
    for (int bit = 63; bit >= 32 + X::low_bits; --bit) settle(bit);
    // the bits that a shorter type lacks are ones below zero, and in a NaN
    constexpr unsigned low = (1u << X::low_bits) - 1u;
    unsigned top = (unsigned)(t >> 32);
    if (!(top & 0x80000000u) || (top | low) == 0xffffffffu) top |= low;
    // as are the upper bits of every place's complement
    const int nb = 32 - __clz((V - 1) | 1);
    t = (unsigned long long)top << 32 | (0x3fffffffu >> nb << nb) << 1;
    for (int bit = nb; bit > 0; --bit) settle(bit);
    __syncthreads();
    if (tid == 0) n_cand = 0;
    __syncthreads();
    each([&](unsigned long long o) {
      if (o >= t) cand[atomicAdd(&n_cand, 1)] = o;
    });
    __syncthreads();
    nc = n_cand;
  }
  // the last wave has the fewest candidates; a row of -inf: log 0
  if (!odd && tid == THREADS - 1)
    lse[r] = (float)((double)s_run.m / temperature + log((double)s_run.s));
  // rank by counting, 8 lanes to a candidate
  for (int i0 = 0; i0 < nc; i0 += THREADS / 8) {
    const int i = i0 + (tid >> 3);
    const unsigned long long mine = i < nc ? cand[i] : ~0ull;
    int rank = 0;
#pragma unroll 4
    for (int q = tid & 7; q < nc; q += 8) rank += cand[q] > mine;
    rank += __builtin_amdgcn_mov_dpp(rank, 0xB1, 15, 15, true);
    rank += __builtin_amdgcn_mov_dpp(rank, 0x4E, 15, 15, true);
    rank += __builtin_amdgcn_mov_dpp(rank, 0x141, 15, 15, true);
    if ((tid & 7) == 0 && i < nc && rank < k) {
      const long long at = (long long)r * k + rank;
      indices[at] = place_of(mine);
      X::put(values + at * X::size, logit_of(mine));
      // a NaN ranks first, and without one the row's +inf is its logsumexp
      if (odd && rank == 0) lse[r] = logit_of(mine);
    }
  }
}

int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// Blocks that a pass asks for at least, splitting rows: 64 rows of 30522 take
// 4.5 us in stats, with 1024 5.8, and as fp32 5.1 in grad, with 2048 6.0; 200
// rows of 128256 14 in stats, with 256 too.
constexpr int kBlocks = 512;

// Splits of a row over blocks: enough blocks to fill the chip, none with less
// than one vector per thread.
int splits_for(const LmRows& in, int seg_most, int* seg) {
  const int per = kThreads * (in.type == LM_FP32 ? 4 : 8);
  int s = div_up(kBlocks, in.R);
  s = std::min(s, std::max(1, div_up(in.V, per)));
  s = std::max(s, div_up(in.V, seg_most));
  // whole vectors per thread, so that segments start where vectors do
  *seg = div_up(div_up(in.V, s), 32) * 32;
  return div_up(in.V, *seg);
}

constexpr long long kMB = 1 << 20;
long long bytes_of(const LmRows& in) {
  return (long long)in.R * in.V * (in.type == LM_FP32 ? 4 : 2);
}

// A segment's most: of stats what its bits in LDS allow; of grad two rounds of
// loads a thread while the cache holds the logits (4096 rows of 30522 fp16 69
// us, in one round 72, in four 71), else one (2048 rows of 128256 150 us, in two
// 155, in four 159, half a round 165).
constexpr int kStatSeg = 131072, kGradSegBytes = 32768, kGradSegFar = 16384;
// Threads of a block of topk: 512, or 1024 where there are no more rows than
// CUs and each is long. At 1024 rows of 128256 both take 56 us (256 threads
// 64), at 4000 rows of 8000 512 take 44 us and 1024 take 72, at 100 rows of
// 262144 33 and 27.
constexpr int kTopkFewRows = 256, kTopkLongRow = 8192;  // vectors

// What the pass over a row leaves in the 256 MB cache behind the L2, the pass
// of the gradient need not fetch again. At 525 MB of logits a cache that every
// line goes through keeps little of them: stats + grad take 97 + 171 us, 83 +
// 166 where all of stats' loads are told not to stay, and 88 + 150 where those
// of 9 rows of 16 may. At 203 MB all may stay (32 + 53 us, else 31 + 66).
constexpr long long kKeepBytes = 300 * kMB;
// A gradient of this size is gone from the caches before anyone reads it, and
// written past them it leaves them the logits: at 244 MB stats + grad take 49 +
// 58 us, else 78 + 72; at 163 MB 33 + 40, else 40 + 55; at 81 MB grad 22, else
// 24. A smaller one stays for the product that follows.
constexpr long long kStreamGrad = 64 * kMB;
// topk reads a row once and its best lines again: streamed at 263 MB 56 against
// 60 us, at 78 MB 22 against 20.
constexpr long long kStreamTopk = 128 * kMB;

int grad_seg(const LmRows& in) {
  return (bytes_of(in) > kKeepBytes ? kGradSegFar : kGradSegBytes) /
         (in.type == LM_FP32 ? 4 : 2);
}

template <int TY>
void grad_of(const LmRows& in, const LmPlaces& pl, const LmKeep& kp,
             const LmUp& up, void* dx, hipStream_t s) {
  int seg;
  const int splits = splits_for(in, grad_seg(in), &seg);
  const dim3 grid((unsigned)in.R * splits);
  const bool nt = bytes_of(in) > kStreamGrad;
  auto kernel = kp.p ? (nt ? lm_grad_kernel<TY, false, true> : lm_grad_kernel<TY, false, false>)
                     : (nt ? lm_grad_kernel<TY, true, true> : lm_grad_kernel<TY, true, false>);
  kernel<<<grid, kThreads, 0, s>>>(in, pl, kp, up, (char*)dx, splits, seg);
}

// Many short rows take a wave each: a block's start, its joins through LDS and
// its end outweigh such a row. This pass alone, again and again: 8192 rows of 600
// bf16 8 us, in blocks of 256 threads 23; 60000 of 5001 112 and 157 (131 behind a
// gradient's pass); 4096 of 16000 24 and 25. A wave alone is
// behind with few rows (512 of 5001 fp32 5.2 and 4.4 us, 1024 of 8200 8.8 and
// 6.8) and with longer ones (8192 of 30522 bf16 with a record 86 and 82).
constexpr int kWaveRows = 2048, kWaveVectors = 2048;

template <int TY, int T>
void stats_with(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
                const LmWork& w, const LmKeep& kp, int splits, int seg,
                hipStream_t s) {
  const dim3 grid((unsigned)in.R * splits + (te.values ? div_up(in.R, T / 64) : 0));
  const int keep16 = (int)std::min(16LL, 16 * kKeepBytes / bytes_of(in));
  const bool top = w.part_top != nullptr;
  auto kernel = top         ? lm_stats_kernel<TY, T, true, true>
                : te.values ? lm_stats_kernel<TY, T, true, false>
                            : lm_stats_kernel<TY, T, false, false>;
  kernel<<<grid, T, top ? ((seg + 31) / 32 + 3) * 4 : 0, s>>>(
      in, pl, te, splits, seg, keep16, w.part, w.part_top, w.xt, kp.p, w.rec,
      w.counter);
}

template <int TY>
void stats_of(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
              const LmWork& w, const LmKeep& kp, hipStream_t s) {
  int seg;
  const int splits = splits_for(in, kStatSeg, &seg);
  if (in.R >= kWaveRows && in.V / Ty<TY>::N <= kWaveVectors)
    stats_with<TY, 64>(in, pl, te, w, kp, splits, seg, s);
  else
    stats_with<TY, kThreads>(in, pl, te, w, kp, splits, seg, s);
}

template <int TY, int T, int PIECE>
void topk_with(const LmRows& in, double temperature, int k, void* values,
               long long* indices, float* lse, hipStream_t s) {
  auto kernel = bytes_of(in) > kStreamTopk ? lm_topk_kernel<TY, T, PIECE, true>
                                           : lm_topk_kernel<TY, T, PIECE, false>;
  kernel<<<dim3(in.R), T, 0, s>>>(in, temperature, k, (char*)values, indices, lse);
}

template <int TY>
void topk_of(const LmRows& in, double temperature, int k, void* values,
             long long* indices, float* lse, hipStream_t s) {
  const int nv = in.V / Ty<TY>::N;
  // lines where there are four of them and more to each of the k
  if (in.V <= kPieces)
    topk_with<TY, 512, kLogits>(in, temperature, k, values, indices, lse, s);
  else if (nv < 32 * k)
    topk_with<TY, 512, kVectors>(in, temperature, k, values, indices, lse, s);
  else if (in.R <= kTopkFewRows && nv > kTopkLongRow)
    topk_with<TY, 1024, kLines>(in, temperature, k, values, indices, lse, s);
  else
    topk_with<TY, 512, kLines>(in, temperature, k, values, indices, lse, s);
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
  return splits_for(in, kStatSeg, &seg);
}

int lm_grad_splits(const LmRows& in) {
  int seg;
  return splits_for(in, grad_seg(in), &seg);
}

int lm_group(int splits) {
  int g = 1;
  while (g < splits && g < 64) g <<= 1;
  return g;
}

// The finish kernels are a chain of latencies: one block where it holds all the
// rows, so that no block waits for another, else blocks of a wave while they
// are few (2048 rows: 6.5 us, in blocks of 256 7.4; 16384 rows 10.6 and 7.4).
static int finish_threads(int R, int group) {
  const long long lanes = (long long)R * group;
  if (lanes <= kThreads) return std::max(64, (int)(lanes + 63) / 64 * 64);
  return lanes <= 8192 ? 64 : kThreads;
}

int lm_finish_blocks(int R, int group) {
  return div_up((long long)R * group, finish_threads(R, group));
}

void lm_distill(const LmRows& in, const LmPlaces& pl, const LmTeacher& te,
                const LmWork& w, const LmKeep& kp, const LmOut& o,
                hipStream_t s) {
  stats(in, pl, te, w, kp, s);
  lm_distill_kernel<<<dim3(lm_finish_blocks(in.R, w.group)),
                      finish_threads(in.R, w.group), 0, s>>>(in, pl, te, w, kp, o);
}

void lm_policy(const LmRows& in, const LmPlaces& pl, const LmPolicy& po,
               const LmWork& w, const LmKeep& kp, float* logps, float* kl,
               const LmOut& o, hipStream_t s) {
  stats(in, pl, LmTeacher{}, w, kp, s);
  lm_policy_kernel<<<dim3(lm_finish_blocks(in.R, w.group)),
                     finish_threads(in.R, w.group), 0, s>>>(in, pl, po, w, kp,
                                                            logps, kl, o);
}

void lm_preference(const LmRows& in, const LmPlaces& pl, const LmPreference& pr,
                   const LmWork& w, const LmKeep& kp, float* chosen,
                   float* rejected, const LmOut& o, hipStream_t s) {
  stats(in, pl, LmTeacher{}, w, kp, s);
  const int pairs = in.R / in.T / 2;
  const long long lanes = 2LL * in.T * w.group;
  const int threads = (int)std::min(1024LL, (lanes + 63) / 64 * 64);
  lm_preference_kernel<<<dim3(pairs), threads, 0, s>>>(in, pl, pr, w, kp, chosen,
                                                       rejected, o);
}

void lm_grad(const LmRows& in, const LmPlaces& pl, const LmKeep& kp,
             const LmUp& up, void* dx, hipStream_t s) {
  LM_BY_TYPE(in.type, (grad_of<TY>(in, pl, kp, up, dx, s)));
}

void lm_topk(const LmRows& in, double temperature, int k, void* values,
             long long* indices, float* lse, hipStream_t s) {
  LM_BY_TYPE(in.type, (topk_of<TY>(in, temperature, k, values, indices, lse, s)));
}
