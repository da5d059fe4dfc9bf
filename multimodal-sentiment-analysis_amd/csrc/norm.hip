// Group normalisation with an activation over channels-last maps x [batch][P positions][C channels], forward and
// backward, in fp32 / bf16 / fp16 (statistics, parameters and their gradients always in 32 bits or more).
//
//   group g of sample b: the N = P * C/G values of its channels;  mean = sum x / N,  var = sum (x - mean)^2 / N,
//   rstd = 1 / sqrt(var + eps),  xhat = (x - mean) rstd,  z = xhat gamma + beta,  y = act(z)
//   dz = dy act'(z),  dgamma = sum_{b,p} dz xhat,  dbeta = sum_{b,p} dz,  q = dz gamma,
//   dx = rstd (q - mean_N(q) - xhat mean_N(q xhat))
//
// A sample is one run of S = P * C values.  Threads walk it in 16-byte vectors of V values; thread t always lands on the
// same V channels because the step of a row of threads is a multiple of lcm(C, V): `period` = C / gcd(C, V) vectors.
// That holds for any C, odd ones too, so there is one code path with 16-byte accesses (a sample may start at any value:
// the vectors are declared with the alignment of one value, which this target's global accesses allow).
#include "mmsa_common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

typedef unsigned u32x4a __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

template <typename T> struct Io;
template <> struct Io<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
  static __device__ __forceinline__ void load(const float* p, float (&o)[4]) {
    const f32x4a r = *reinterpret_cast<const f32x4a*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = r[i];
  }
  static __device__ __forceinline__ void store(float* p, const float (&o)[4]) {
    f32x4a r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = o[i];
    *reinterpret_cast<f32x4a*>(p) = r;
  }
};
// 16-bit values travel as raw bits
__device__ __forceinline__ float bf16_to_f32(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float f) {
  __hip_bfloat16 h = __float2bfloat16(f);   // round to nearest even
  unsigned short u;
  __builtin_memcpy(&u, &h, 2);
  return u;
}
struct bf16_t { unsigned short b; };
struct fp16_t { _Float16 h; };
template <> struct Io<bf16_t> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float to(bf16_t v) { return bf16_to_f32(v.b); }
  static __device__ __forceinline__ bf16_t from(float v) { return bf16_t{f32_to_bf16(v)}; }
  static __device__ __forceinline__ void load(const bf16_t* p, float (&o)[8]) {
    const u32x4a r = *reinterpret_cast<const u32x4a*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(r[i] << 16);
      o[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float (&o)[8]) {
    u32x4a r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (unsigned)f32_to_bf16(o[2 * i]) | ((unsigned)f32_to_bf16(o[2 * i + 1]) << 16);
    *reinterpret_cast<u32x4a*>(p) = r;
  }
};
template <> struct Io<fp16_t> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float to(fp16_t v) { return (float)v.h; }
  static __device__ __forceinline__ fp16_t from(float v) { return fp16_t{(_Float16)v}; }
  static __device__ __forceinline__ void load(const fp16_t* p, float (&o)[8]) {
    const u32x4a r = *reinterpret_cast<const u32x4a*>(p);
    _Float16 h[8];
    __builtin_memcpy(h, &r, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)h[i];
  }
  static __device__ __forceinline__ void store(fp16_t* p, const float (&o)[8]) {
    _Float16 h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)o[i];
    u32x4a r;
    __builtin_memcpy(&r, h, 16);
    *reinterpret_cast<u32x4a*>(p) = r;
  }
};

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
  if (ACT == ACT_SILU) return z / (1.f + __expf(-z));
  if (ACT == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (ACT == ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-z));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == ACT_GELU)
    return fmaf(z * 0.39894228040143268f, __expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
  return 1.f;
}

// How a sample is cut: `active` threads of a block cover rows of `active` vectors (a multiple of the period), `columns`
// of them one after another where the period is longer than a block; a chunk is `iters` such rows.
struct Cut {
  long S;          // values per sample
  long nvec;       // vectors per sample, the last one possibly cut short
  int C, G, Cg;
  int period, active, columns;
  int row;         // vectors from one row of threads to the next (active where columns == 1, else period)
  int iters;
  long nchunk;     // chunks per sample
};

// ---------------------------------------------------------------------------------------------------- statistics
// Every thread sums d = x - k and d^2 per channel, k being its own first value: as k is one of the values summed, the
// sum of squares about the thread's mean loses at most a few roundings to cancellation, whatever the mean of the map
// is.  Threads, chunks and channels are then joined in 64 bits by the parallel-variance formula
//   M2 = sum M2_i + sum n_i (mean_i - mean)^2.
template <typename T>
__global__ __launch_bounds__(1024) void gn_stats_kernel(const T* __restrict__ x, const Cut cut,
                                                        double* __restrict__ part) {
  constexpr int V = Io<T>::V;
  extern __shared__ float sh[];                 // [3][slots]: mean, M2, count of every (thread, element)
  const int tid = threadIdx.x;
  const long b = blockIdx.x / cut.nchunk, ch = blockIdx.x % cut.nchunk;
  const T* xs = x + b * cut.S;
  const int slots = cut.columns == 1 ? cut.active * V : cut.period * V;
  float* smean = sh;
  float* sm2 = sh + slots;
  float* scnt = sh + 2 * slots;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    float k[V], s[V], q[V];
    int cnt[V];
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f, cnt[e] = 0;
    const long v0 = ch * cut.iters * (long)cut.row + t;
    for (int it = 0; it < cut.iters; ++it) {
      const long v = v0 + it * (long)cut.row;
      if (v >= cut.nvec) break;
      const long at = v * V;
      float f[V];
      if (at + V <= cut.S) {
        Io<T>::load(xs + at, f);
        if (it == 0) {
#pragma unroll
          for (int e = 0; e < V; ++e) k[e] = f[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = f[e] - k[e];
          s[e] += d;
          q[e] = fmaf(d, d, q[e]);
          ++cnt[e];
        }
      } else {
        for (int e = 0; e < (int)(cut.S - at); ++e) {
          const float fe = Io<T>::to(xs[at + e]);
          if (it == 0) k[e] = fe;
          const float d = fe - k[e];
          s[e] += d;
          q[e] = fmaf(d, d, q[e]);
          ++cnt[e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float n = (float)cnt[e];
      const float m = cnt[e] ? s[e] / n : 0.f;
      smean[t * V + e] = k[e] + m;
      sm2[t * V + e] = fmaxf(fmaf(-s[e], m, q[e]), 0.f);
      scnt[t * V + e] = n;
    }
  }
  __syncthreads();
  // one wave per group, round robin; slot q belongs to channel q % C (slots is a multiple of C)
  const int lane = tid & 63, w = tid >> 6, nw = blockDim.x >> 6;
  const int reps = slots / cut.C;
  const int per = reps * cut.Cg;
  for (int g = w; g < cut.G; g += nw) {
    double n = 0.0, sum = 0.0;
    for (int i = lane; i < per; i += 64) {
      const int q = (i / cut.Cg) * cut.C + g * cut.Cg + i % cut.Cg;
      n += (double)scnt[q];
      sum += (double)scnt[q] * (double)smean[q];
    }
    n = wave_sum_d(n);
    sum = wave_sum_d(sum);
    const double mean = n > 0.0 ? sum / n : 0.0;
    double m2 = 0.0;
    for (int i = lane; i < per; i += 64) {
      const int q = (i / cut.Cg) * cut.C + g * cut.Cg + i % cut.Cg;
      const double d = (double)smean[q] - mean;
      if (scnt[q] > 0.f) m2 += (double)sm2[q] + (double)scnt[q] * d * d;
    }
    m2 = wave_sum_d(m2);
    if (lane == 0) {
      double* o = part + ((long)blockIdx.x * cut.G + g) * 3;
      o[0] = n;
      o[1] = mean;
      o[2] = m2;
    }
  }
}

// joins the chunks of one (sample, group): one wave each
__global__ __launch_bounds__(64) void gn_stats_join_kernel(const double* __restrict__ part, long nchunk, int G,
                                                           float eps, double* __restrict__ stats) {
  const long b = blockIdx.x / G;
  const int g = blockIdx.x % G, lane = threadIdx.x;
  const double* p = part + (b * nchunk * G + g) * 3;
  const long step = (long)G * 3;
  double n = 0.0, sum = 0.0;
  for (long i = lane; i < nchunk; i += 64) {
    n += p[i * step];
    sum += p[i * step] * p[i * step + 1];
  }
  n = wave_sum_d(n);
  sum = wave_sum_d(sum);
  const double mean = sum / n;
  double m2 = 0.0;
  for (long i = lane; i < nchunk; i += 64) {
    const double d = p[i * step + 1] - mean;
    m2 += p[i * step + 2] + p[i * step] * d * d;
  }
  m2 = wave_sum_d(m2);
  if (lane == 0) {
    stats[2 * blockIdx.x] = mean;
    stats[2 * blockIdx.x + 1] = 1.0 / sqrt(m2 / n + (double)eps);
  }
}

// ---------------------------------------------------------------------------------------------------- forward map
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_apply_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                        const float* __restrict__ beta,
                                                        const double* __restrict__ stats, T* __restrict__ y,
                                                        const Cut cut) {
  constexpr int V = Io<T>::V;
  const int tid = threadIdx.x;
  const long b = blockIdx.x / cut.nchunk, ch = blockIdx.x % cut.nchunk;
  const T* xs = x + b * cut.S;
  T* ys = y + b * cut.S;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    float mean[V], a[V], o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (int)(((long)t * V + e) % cut.C);
      const double* st = stats + 2 * (b * cut.G + c / cut.Cg);
      mean[e] = (float)st[0];
      a[e] = (float)st[1] * (gamma ? gamma[c] : 1.f);
      o[e] = beta ? beta[c] : 0.f;
    }
    const long v0 = ch * cut.iters * (long)cut.row + t;
    for (int it = 0; it < cut.iters; ++it) {
      const long v = v0 + it * (long)cut.row;
      if (v >= cut.nvec) break;
      const long at = v * V;
      float f[V];
      if (at + V <= cut.S) {
        Io<T>::load(xs + at, f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = act_fwd<ACT>(fmaf(f[e] - mean[e], a[e], o[e]));
        Io<T>::store(ys + at, f);
      } else {
        for (int e = 0; e < (int)(cut.S - at); ++e)
          ys[at + e] = Io<T>::from(act_fwd<ACT>(fmaf(Io<T>::to(xs[at + e]) - mean[e], a[e], o[e])));
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------- backward
// The slope of the activation at z.  Which side of zero a ReLU's input lies on decides a whole gradient element, so
// where the 32-bit z is within its own rounding of zero the decision is made in 64 bits from the 64-bit statistics.
template <int ACT>
__device__ __forceinline__ float gn_slope(float x, float xh, float gam, float bet, const double* __restrict__ st) {
  const float z = fmaf(xh, gam, bet);
  if (ACT == ACT_RELU) {
    const float mr = fabsf((float)(st[0] * st[1]));
    if (fabsf(z) <= 3.8e-6f * (fabsf(gam) * (fabsf(xh) + mr) + fabsf(bet)))
      return ((double)x - st[0]) * st[1] * (double)gam + (double)bet > 0.0 ? 1.f : 0.f;
  }
  return act_slope<ACT>(z);
}

// per chunk and channel: sum of dz and of dz xhat
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                           const float* __restrict__ gamma,
                                                           const float* __restrict__ beta,
                                                           const double* __restrict__ stats, const Cut cut,
                                                           float* __restrict__ part) {
  constexpr int V = Io<T>::V;
  extern __shared__ float sh[];
  const int tid = threadIdx.x;
  const long b = blockIdx.x / cut.nchunk, ch = blockIdx.x % cut.nchunk;
  const T* xs = x + b * cut.S;
  const T* gs = dy + b * cut.S;
  const int slots = cut.columns == 1 ? cut.active * V : cut.period * V;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    float mean[V], rstd[V], gam[V], bet[V], s1[V], s2[V];
    const double* st[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (int)(((long)t * V + e) % cut.C);
      st[e] = stats + 2 * (b * cut.G + c / cut.Cg);
      mean[e] = (float)st[e][0];
      rstd[e] = (float)st[e][1];
      gam[e] = gamma ? gamma[c] : 1.f;
      bet[e] = beta ? beta[c] : 0.f;
      s1[e] = s2[e] = 0.f;
    }
    const long v0 = ch * cut.iters * (long)cut.row + t;
    for (int it = 0; it < cut.iters; ++it) {
      const long v = v0 + it * (long)cut.row;
      if (v >= cut.nvec) break;
      const long at = v * V;
      float f[V], d[V];
      if (at + V <= cut.S) {
        Io<T>::load(xs + at, f);
        Io<T>::load(gs + at, d);
      } else {
        for (int e = 0; e < V; ++e) {
          const bool in = at + e < cut.S;
          f[e] = in ? Io<T>::to(xs[at + e]) : 0.f;
          d[e] = in ? Io<T>::to(gs[at + e]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (f[e] - mean[e]) * rstd[e];
        const float dz = d[e] * gn_slope<ACT>(f[e], xh, gam[e], bet[e], st[e]);
        s1[e] += dz;
        s2[e] = fmaf(dz, xh, s2[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sh[t * V + e] = s1[e];
      sh[slots + t * V + e] = s2[e];
    }
  }
  __syncthreads();
  for (int c = tid; c < cut.C; c += blockDim.x) {
    float a = 0.f, q = 0.f;
    for (int r = c; r < slots; r += cut.C) {
      a += sh[r];
      q += sh[slots + r];
    }
    float* o = part + ((long)blockIdx.x * cut.C + c) * 2;
    o[0] = a;
    o[1] = q;
  }
}

// joins the chunks of one (sample, group): channel sums [b][c][2], and the two means of the group over N values
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(const float* __restrict__ part, const Cut cut,
                                                          const float* __restrict__ gamma, float* __restrict__ sums,
                                                          float* __restrict__ coef) {
  __shared__ double red[16];
  const long b = blockIdx.x / cut.G;
  const int g = blockIdx.x % cut.G, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double c1 = 0.0, c2 = 0.0;
  for (int j = w; j < cut.Cg; j += 4) {           // one wave per channel
    const int c = g * cut.Cg + j;
    const float* p = part + (b * cut.nchunk * cut.C + c) * 2;
    double a = 0.0, q = 0.0;
    for (long i = lane; i < cut.nchunk; i += 64) {
      a += (double)p[i * cut.C * 2];
      q += (double)p[i * cut.C * 2 + 1];
    }
    a = wave_sum_d(a);
    q = wave_sum_d(q);
    if (lane == 0) {
      sums[(b * cut.C + c) * 2] = (float)a;
      sums[(b * cut.C + c) * 2 + 1] = (float)q;
      const double gm = gamma ? (double)gamma[c] : 1.0;
      c1 += a * gm;
      c2 += q * gm;
    }
  }
  c1 = block_sum_d(c1, red);
  c2 = block_sum_d(c2, red);
  if (threadIdx.x == 0) {
    const double n = (double)(cut.S / cut.C) * cut.Cg;
    coef[2 * blockIdx.x] = (float)(c1 / n);
    coef[2 * blockIdx.x + 1] = (float)(c2 / n);
  }
}

// blocks [0, nparam): dgamma / dbeta, a channel per thread, summed over the samples in order; the others: dx
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                            const float* __restrict__ gamma,
                                                            const float* __restrict__ beta,
                                                            const double* __restrict__ stats,
                                                            const float* __restrict__ sums,
                                                            const float* __restrict__ coef, T* __restrict__ dx,
                                                            float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                            int nparam, long batch, const Cut cut) {
  constexpr int V = Io<T>::V;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < nparam) {
    const int c = blockIdx.x * blockDim.x + tid;
    if (c >= cut.C) return;
    double a = 0.0, q = 0.0;
    for (long b = 0; b < batch; ++b) {
      a += (double)sums[(b * cut.C + c) * 2];
      q += (double)sums[(b * cut.C + c) * 2 + 1];
    }
    if (dbeta) dbeta[c] = (float)a;
    if (dgamma) dgamma[c] = (float)q;
    return;
  }
  const long blk = (long)blockIdx.x - nparam;
  const long b = blk / cut.nchunk, ch = blk % cut.nchunk;
  const T* xs = x + b * cut.S;
  const T* gs = dy + b * cut.S;
  T* os = dx + b * cut.S;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    float mean[V], rstd[V], gam[V], bet[V], k1[V], k2[V];
    const double* st[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (int)(((long)t * V + e) % cut.C);
      const long bg = b * cut.G + c / cut.Cg;
      st[e] = stats + 2 * bg;
      mean[e] = (float)st[e][0];
      rstd[e] = (float)st[e][1];
      gam[e] = gamma ? gamma[c] : 1.f;
      bet[e] = beta ? beta[c] : 0.f;
      k1[e] = coef[2 * bg];
      k2[e] = coef[2 * bg + 1];
    }
    const long v0 = ch * cut.iters * (long)cut.row + t;
    for (int it = 0; it < cut.iters; ++it) {
      const long v = v0 + it * (long)cut.row;
      if (v >= cut.nvec) break;
      const long at = v * V;
      const bool whole = at + V <= cut.S;
      float f[V], d[V];
      if (whole) {
        Io<T>::load(xs + at, f);
        Io<T>::load(gs + at, d);
      } else {
        for (int e = 0; e < V; ++e) {
          const bool in = at + e < cut.S;
          f[e] = in ? Io<T>::to(xs[at + e]) : 0.f;
          d[e] = in ? Io<T>::to(gs[at + e]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (f[e] - mean[e]) * rstd[e];
        const float q = d[e] * gn_slope<ACT>(f[e], xh, gam[e], bet[e], st[e]) * gam[e];
        f[e] = rstd[e] * (q - fmaf(xh, k2[e], k1[e]));
      }
      if (whole) {
        Io<T>::store(os + at, f);
      } else {
        for (int e = 0; e < (int)(cut.S - at); ++e) os[at + e] = Io<T>::from(f[e]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------- host side
constexpr int GN_MAX_CHANNELS = 4096;
constexpr int GN_MAX_SLOTS = 12288;         // three floats of LDS for each: 144 of the 160 KiB
constexpr long GN_MAX_BLOCKS = 4000000;     // a grid's threads are counted in 32 bits, blocks have up to 1024

int value_lanes(int dtype) { return dtype == 0 ? 4 : 8; }

bool make_cut(long batch, long positions, int C, int G, int dtype, Cut* cut) {
  if (batch < 1 || positions < 1 || C < 1 || G < 1 || C % G || dtype < 0 || dtype > 2) return false;
  const int V = value_lanes(dtype);
  cut->C = C;
  cut->G = G;
  cut->Cg = C / G;
  cut->S = positions * C;
  cut->nvec = (cut->S + V - 1) / V;
  int a = C, b = V;
  while (b) {
    const int r = a % b;
    a = b;
    b = r;
  }
  cut->period = C / a;
  if (cut->period <= 256) {
    cut->active = cut->period * (256 / cut->period);
    cut->columns = 1;
    cut->row = cut->active;
  } else if (cut->period <= 1024) {
    cut->active = cut->row = cut->period;
    cut->columns = 1;
  } else {
    cut->active = 1024;
    cut->columns = (cut->period + 1023) / 1024;
    cut->row = cut->period;
  }
  const long rows = (cut->nvec + cut->row - 1) / cut->row;
  // chunks: about eight blocks for every compute unit over the whole batch, at least four rows each
  long iters = (rows * batch + 2047) / 2048;
  if (iters < 4) iters = 4;
  if (iters > rows) iters = rows;
  cut->iters = (int)iters;
  cut->nchunk = (rows + iters - 1) / iters;
  return true;
}

int block_of(const Cut& cut) { return (cut.active + 63) / 64 * 64; }
size_t slots_of(const Cut& cut, int dtype) {
  return (size_t)(cut.columns == 1 ? cut.active : cut.period) * value_lanes(dtype);
}
// dynamic LDS of the sums kernels: a block's (thread, value) slots; at most 12 * GN_MAX_SLOTS bytes
template <typename K>
int allow_lds(K kernel, size_t bytes) {
  static PerDeviceOnce once;
  if (bytes > 65536 && once.pending()) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                            160 * 1024) != hipSuccess)
      return MMSA_ERR_LAUNCH;
    once.done();
  }
  return MMSA_OK;
}

template <typename T>
int gn_fwd(const void* x, const float* gamma, const float* beta, void* y, double* stats, void* scratch, long batch,
           const Cut& cut, int dtype, float eps, int act, hipStream_t s) {
  const T* xp = static_cast<const T*>(x);
  T* yp = static_cast<T*>(y);
  const dim3 grid((unsigned)(batch * cut.nchunk)), block(block_of(cut));
  const size_t lds = 3 * sizeof(float) * slots_of(cut, dtype);
  if (int rc = allow_lds(gn_stats_kernel<T>, lds)) return rc;
  hipLaunchKernelGGL((gn_stats_kernel<T>), grid, block, lds, s, xp, cut, static_cast<double*>(scratch));
  hipLaunchKernelGGL(gn_stats_join_kernel, dim3((unsigned)(batch * cut.G)), dim3(64), 0, s,
                     static_cast<const double*>(scratch), cut.nchunk, cut.G, eps, stats);
#define GN_APPLY(A) \
  hipLaunchKernelGGL((gn_apply_kernel<T, A>), grid, block, 0, s, xp, gamma, beta, stats, yp, cut)
  switch (act) {
    case ACT_NONE: GN_APPLY(ACT_NONE); break;
    case ACT_RELU: GN_APPLY(ACT_RELU); break;
    case ACT_SILU: GN_APPLY(ACT_SILU); break;
    default: GN_APPLY(ACT_GELU); break;
  }
#undef GN_APPLY
  return mmsa_launch_status();
}

template <typename T, int ACT>
int gn_bwd(const void* dy, const void* x, const float* gamma, const float* beta, const double* stats, void* dx,
           float* dgamma, float* dbeta, void* scratch, long batch, const Cut& cut, int dtype, hipStream_t s) {
  const T* xp = static_cast<const T*>(x);
  const T* gp = static_cast<const T*>(dy);
  float* part = static_cast<float*>(scratch);
  float* sums = part + batch * cut.nchunk * cut.C * 2;
  float* coef = sums + batch * cut.C * 2;
  const dim3 grid((unsigned)(batch * cut.nchunk)), block(block_of(cut));
  const size_t lds = 2 * sizeof(float) * slots_of(cut, dtype);
  if (int rc = allow_lds(gn_bwd_sums_kernel<T, ACT>, lds)) return rc;
  hipLaunchKernelGGL((gn_bwd_sums_kernel<T, ACT>), grid, block, lds, s, gp, xp, gamma, beta, stats, cut, part);
  hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)(batch * cut.G)), dim3(256), 0, s, part, cut, gamma, sums, coef);
  const int nparam = dgamma || dbeta ? mmsa_cdiv(cut.C, block.x) : 0;
  const unsigned blocks = nparam + (dx ? grid.x : 0);
  if (blocks)
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, ACT>), dim3(blocks), block, 0, s, gp, xp, gamma, beta, stats, sums, coef,
                       static_cast<T*>(dx), dgamma, dbeta, nparam, batch, cut);
  return mmsa_launch_status();
}

template <typename T>
int gn_bwd_act(int act, const void* dy, const void* x, const float* gamma, const float* beta, const double* stats,
               void* dx, float* dgamma, float* dbeta, void* scratch, long batch, const Cut& cut, int dtype,
               hipStream_t s) {
  switch (act) {
    case ACT_NONE:
      return gn_bwd<T, ACT_NONE>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
    case ACT_RELU:
      return gn_bwd<T, ACT_RELU>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
    case ACT_SILU:
      return gn_bwd<T, ACT_SILU>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
    default:
      return gn_bwd<T, ACT_GELU>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
  }
}

int check_size(long batch, long positions, int channels, int groups, int dtype, Cut* cut) {
  if (!make_cut(batch, positions, channels, groups, dtype, cut)) return MMSA_ERR_ARG;
  if (channels > GN_MAX_CHANNELS || slots_of(*cut, dtype) > GN_MAX_SLOTS) return MMSA_ERR_LIMIT;
  if (batch > GN_MAX_BLOCKS / cut->nchunk || batch > 4 * GN_MAX_BLOCKS / groups) return MMSA_ERR_LIMIT;
  return MMSA_OK;
}

}  // namespace

// Bytes of scratch either direction needs for these sizes (the larger of the two; 8-byte aligned).
MMSA_EXPORT long mmsa_group_norm_act_scratch_bytes(long batch, long positions, int channels, int groups, int dtype) {
  Cut cut;
  if (int rc = check_size(batch, positions, channels, groups, dtype, &cut)) return rc;
  const long fwd = batch * cut.nchunk * groups * 3 * 8;
  const long bwd = (batch * cut.nchunk * channels + batch * channels + batch * groups) * 2 * 4;
  return fwd > bwd ? fwd : bwd;
}

// y = act(group_norm(x) gamma + beta); stats [batch][groups][2] <- mean, 1 / sqrt(var + eps) in double
MMSA_EXPORT int mmsa_group_norm_act_fwd(const void* x, const float* gamma, const float* beta, void* y, double* stats,
                                        void* scratch, long batch, long positions, int channels, int groups, float eps,
                                        int act, int dtype, void* stream) {
  MMSA_REQUIRE(x && y && stats && scratch && act >= 0 && act <= 3 && eps >= 0.f);
  Cut cut;
  if (int rc = check_size(batch, positions, channels, groups, dtype, &cut)) return rc;
  hipStream_t s = mmsa_stream(stream);
  if (dtype == 0) return gn_fwd<float>(x, gamma, beta, y, stats, scratch, batch, cut, dtype, eps, act, s);
  if (dtype == 1) return gn_fwd<bf16_t>(x, gamma, beta, y, stats, scratch, batch, cut, dtype, eps, act, s);
  return gn_fwd<fp16_t>(x, gamma, beta, y, stats, scratch, batch, cut, dtype, eps, act, s);
}

// Gradients of mmsa_group_norm_act_fwd; dx, dgamma, dbeta may each be null (not wanted).
MMSA_EXPORT int mmsa_group_norm_act_bwd(const void* dy, const void* x, const float* gamma, const float* beta,
                                        const double* stats, void* dx, float* dgamma, float* dbeta, void* scratch,
                                        long batch, long positions, int channels, int groups, int act, int dtype,
                                        void* stream) {
  MMSA_REQUIRE(dy && x && stats && scratch && act >= 0 && act <= 3);
  Cut cut;
  if (int rc = check_size(batch, positions, channels, groups, dtype, &cut)) return rc;
  hipStream_t s = mmsa_stream(stream);
  if (dtype == 0)
    return gn_bwd_act<float>(act, dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
  if (dtype == 1)
    return gn_bwd_act<bf16_t>(act, dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
  return gn_bwd_act<fp16_t>(act, dy, x, gamma, beta, stats, dx, dgamma, dbeta, scratch, batch, cut, dtype, s);
}
