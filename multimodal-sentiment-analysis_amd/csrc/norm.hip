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

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

typedef unsigned u32x4a __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2a __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u32a __attribute__((aligned(2)));

// 16-bit values travel as raw bits
struct bf16_t { unsigned short b; };
struct fp16_t { _Float16 h; };
__device__ __forceinline__ unsigned short f32_to_bf16(float f) {
  const __bf16 h = (__bf16)f;               // round to nearest even, one conversion instruction for two values
  unsigned short u;
  __builtin_memcpy(&u, &h, 2);
  return u;
}
template <typename T> struct Io;
template <> struct Io<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Io<bf16_t> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float to(bf16_t v) { return __uint_as_float((unsigned)v.b << 16); }
  static __device__ __forceinline__ bf16_t from(float v) { return bf16_t{f32_to_bf16(v)}; }
};
template <> struct Io<fp16_t> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float to(fp16_t v) { return (float)v.h; }
  static __device__ __forceinline__ fp16_t from(float v) { return fp16_t{(_Float16)v}; }
};

// W values as they lie in memory (2 to 16 bytes), and their 32-bit values
template <int BYTES> struct Bits;
template <> struct Bits<16> { typedef u32x4a type; };
template <> struct Bits<8> { typedef u32x2a type; };
template <> struct Bits<4> { typedef u32a type; };
template <> struct Bits<2> { typedef unsigned short type; };
template <typename T, int W> struct Pack {
  typename Bits<W * (int)sizeof(T)>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const decltype(raw)*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<decltype(raw)*>(p) = raw; }
  __device__ __forceinline__ void get(float (&o)[W]) const {
    T v[W];
    __builtin_memcpy(v, &raw, W * sizeof(T));
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] = Io<T>::to(v[i]);
  }
  __device__ __forceinline__ void set(const float (&o)[W]) {
    T v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = Io<T>::from(o[i]);
    __builtin_memcpy(&raw, v, W * sizeof(T));
  }
};

// The kernels on 16-bit maps are bound by the vector unit as much as by memory, so the activations are written for few
// instructions: the hardware's exponential and reciprocal (each good to about 1 unit of float32), and for GELU
//   Phi(z) = 1 - e P(t) for z >= 0, e P(t) for z < 0,  e = exp(-z^2 / 2),  t = 1 / (1 + p |z| / sqrt 2)
// (Abramowitz and Stegun 7.1.26, 0.75e-7 off at most), which shares its exponential with the density in the slope.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-z)); }
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  e = fast_exp(-0.5f * z * z);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
  float p = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  p = fmaf(t, p, 0.5f * 1.421413741f);
  p = fmaf(t, p, 0.5f * -0.284496736f);
  p = fmaf(t, p, 0.5f * 0.254829592f);
  p *= t * e;
  return z < 0.f ? p : 1.f - p;
}
template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
  if (ACT == ACT_SILU) return z * sigmoid(z);
  if (ACT == ACT_GELU) {
    float e;
    return z * normal_cdf(z, e);
  }
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == ACT_GELU) {
    float e;
    const float c = normal_cdf(z, e);
    return fmaf(z * 0.39894228040143268f, e, c);
  }
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
  int team;        // lanes that join the statistics of a group, a power of two up to a wave
};

// sum over aligned teams of `team` lanes, the same in every lane of a team
__device__ __forceinline__ double team_sum(double v, int team) {
  for (int s = 1; s < team; s <<= 1) v += __shfl_xor(v, s);
  return v;
}

// a thread's share of a chunk: `full` whole vectors, `row` apart, from the first on; then possibly the sample's last,
// shorter one
struct Share {
  long at;      // first value
  int full;
  int rest;     // values of the short vector behind them, 0: none
};
template <int V>
__device__ __forceinline__ Share share_of(const Cut& cut, long ch, int t) {
  const long v0 = ch * cut.iters * (long)cut.row + t, whole = cut.S / V;
  Share s;
  s.at = v0 * V;
  long n = v0 < whole ? (whole - v0 + cut.row - 1) / cut.row : 0;
  if (n > cut.iters) n = cut.iters;
  s.full = (int)n;
  s.rest = n < cut.iters && v0 + n * cut.row == whole ? (int)(cut.S - whole * V) : 0;
  return s;
}

// ---------------------------------------------------------------------------------------------------- statistics
// Every thread sums d = x - k and d^2 per channel, k being its own first value: as k is one of the values summed, the
// sum of squares about the thread's mean loses at most a few roundings to cancellation, whatever the mean of the map
// is.  Threads, chunks and channels are then joined in 64 bits by the parallel-variance formula
//   M2 = sum M2_i + sum n_i (mean_i - mean)^2.
template <typename T>
__global__ __launch_bounds__(1024) void gn_stats_kernel(const T* __restrict__ x, const Cut cut,
                                                        double* __restrict__ part) {
  constexpr int V = Io<T>::V, U = 4;            // U loads in flight per thread
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
    const Share me = share_of<V>(cut, ch, t);
    const T* p = xs + me.at;
    const long hop = (long)cut.row * V;
    float k[V], s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
    if (me.full) {
      Pack<T, V> f;
      f.load(p);
      f.get(k);
    }
    int it = 0;
    for (; it + U <= me.full; it += U, p += U * hop) {
      Pack<T, V> f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u].load(p + u * hop);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[V];
        f[u].get(v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = v[e] - k[e];
          s[e] += d;
          q[e] = fmaf(d, d, q[e]);
        }
      }
    }
    for (; it < me.full; ++it, p += hop) {
      Pack<T, V> f;
      f.load(p);
      float v[V];
      f.get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = v[e] - k[e];
        s[e] += d;
        q[e] = fmaf(d, d, q[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (e < me.rest) {
        const float v = Io<T>::to(p[e]);
        if (!me.full) k[e] = v;
        const float d = v - k[e];
        s[e] += d;
        q[e] = fmaf(d, d, q[e]);
      }
      const float n = (float)(me.full + (e < me.rest ? 1 : 0));
      const float m = n > 0.f ? s[e] / n : 0.f;
      smean[t * V + e] = k[e] + m;
      sm2[t * V + e] = fmaxf(fmaf(-s[e], m, q[e]), 0.f);
      scnt[t * V + e] = n;
    }
  }
  __syncthreads();
  // a team of lanes per group, all groups at once where there are enough threads; slot q belongs to channel q % C
  // (slots is a multiple of C)
  const int per = slots / cut.C * cut.Cg;
  const int lane = tid & (cut.team - 1), teams = blockDim.x / cut.team;
  for (int g0 = 0; g0 < cut.G; g0 += teams) {          // uniform: all lanes take part in the sums
    const int g = g0 + tid / cut.team;
    const bool mine = g < cut.G;
    double n = 0.0, sum = 0.0;
    for (int i = lane; mine && i < per; i += cut.team) {
      const int q = (i / cut.Cg) * cut.C + g * cut.Cg + i % cut.Cg;
      n += (double)scnt[q];
      sum += (double)scnt[q] * (double)smean[q];
    }
    n = team_sum(n, cut.team);
    sum = team_sum(sum, cut.team);
    const double mean = n > 0.0 ? sum / n : 0.0;
    double m2 = 0.0;
    for (int i = lane; mine && i < per; i += cut.team) {
      const int q = (i / cut.Cg) * cut.C + g * cut.Cg + i % cut.Cg;
      const double d = (double)smean[q] - mean;
      if (scnt[q] > 0.f) m2 += (double)sm2[q] + (double)scnt[q] * d * d;
    }
    m2 = team_sum(m2, cut.team);
    if (mine && lane == 0) {
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
// (The chunks are taken in reverse order: what the statistics pass read last is still in the cache.)
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_apply_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                        const float* __restrict__ beta,
                                                        const double* __restrict__ stats, T* __restrict__ y,
                                                        const Cut cut) {
  constexpr int V = Io<T>::V, U = 4;
  const int tid = threadIdx.x;
  const long blk = (long)gridDim.x - 1 - blockIdx.x, b = blk / cut.nchunk, ch = blk % cut.nchunk;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    const Share me = share_of<V>(cut, ch, t);
    if (me.full + me.rest == 0) continue;
    const T* p = x + b * cut.S + me.at;
    T* o = y + b * cut.S + me.at;
    const long hop = (long)cut.row * V;
    float mean[V], a[V], c0[V];
    int c = (int)(((long)t * V) % cut.C);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const double* st = stats + 2 * (b * cut.G + c / cut.Cg);
      mean[e] = (float)st[0];
      a[e] = (float)st[1] * (gamma ? gamma[c] : 1.f);
      c0[e] = beta ? beta[c] : 0.f;
      if (++c == cut.C) c = 0;
    }
    auto map = [&](Pack<T, V>& f) {
      float v[V];
      f.get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = act_fwd<ACT>(fmaf(v[e] - mean[e], a[e], c0[e]));
      f.set(v);
    };
    int it = 0;
    for (; it + U <= me.full; it += U, p += U * hop, o += U * hop) {
      Pack<T, V> f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u].load(p + u * hop);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        map(f[u]);
        f[u].store(o + u * hop);
      }
    }
    for (; it < me.full; ++it, p += hop, o += hop) {
      Pack<T, V> f;
      f.load(p);
      map(f);
      f.store(o);
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < me.rest) o[e] = Io<T>::from(act_fwd<ACT>(fmaf(Io<T>::to(p[e]) - mean[e], a[e], c0[e])));
  }
}

// ---------------------------------------------------------------------------------------------------- backward
// what a thread knows of the channels of its V values: z = (x - mean) a + beta with a = gamma rstd
template <int V>
struct Channel {
  float mean[V], a[V], bet[V];
  int c, C, Cg;
  const float* gamma;
  const double* stats;      // of the sample
  __device__ __forceinline__ void load(const double* st, const float* gam, const float* beta, int first, int channels,
                                       int per_group) {
    c = first;
    C = channels;
    Cg = per_group;
    gamma = gam;
    stats = st;
    int k = first;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      mean[e] = (float)st[2 * (k / Cg)];
      a[e] = (float)st[2 * (k / Cg) + 1] * (gam ? gam[k] : 1.f);
      bet[e] = beta ? beta[k] : 0.f;
      if (++k == C) k = 0;
    }
  }
  // d = x - mean and the slope of the activation there.  Which side of zero a ReLU's input lies on decides a whole
  // gradient element, so where the 32-bit z is within its own rounding of zero the decision is made in 64 bits from the
  // 64-bit statistics.
  template <int ACT>
  __device__ __forceinline__ float slope(int e, float x, float& d) const {
    d = x - mean[e];
    const float z = fmaf(d, a[e], bet[e]);
    if (ACT == ACT_RELU) {
      if (fabsf(z) <= 3.8e-6f * (fabsf(a[e]) * (fabsf(d) + fabsf(mean[e])) + fabsf(bet[e]))) {
        const int k = (c + e) % C;
        const double* st = stats + 2 * (k / Cg);
        return ((double)x - st[0]) * st[1] * (gamma ? (double)gamma[k] : 1.0) + (double)bet[e] > 0.0 ? 1.f : 0.f;
      }
    }
    return act_slope<ACT>(z);
  }
};

// per chunk and channel: sum of dz and of dz xhat
template <typename T, int ACT>
__global__ __launch_bounds__(1024) void gn_bwd_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                           const float* __restrict__ gamma,
                                                           const float* __restrict__ beta,
                                                           const double* __restrict__ stats, const Cut cut,
                                                           float* __restrict__ part) {
  constexpr int V = Io<T>::V, U = 2;
  extern __shared__ float sh[];
  const int tid = threadIdx.x;
  const long b = blockIdx.x / cut.nchunk, ch = blockIdx.x % cut.nchunk;
  const int slots = cut.columns == 1 ? cut.active * V : cut.period * V;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    const Share me = share_of<V>(cut, ch, t);
    const T* p = x + b * cut.S + me.at;
    const T* g = dy + b * cut.S + me.at;
    const long hop = (long)cut.row * V;
    Channel<V> k;
    k.load(stats + 2 * b * cut.G, gamma, beta, (int)(((long)t * V) % cut.C), cut.C, cut.Cg);
    float s1[V], s2[V];           // sums of dz and of dz (x - mean)
#pragma unroll
    for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
    auto add = [&](int e, float v, float h) {
      float d;
      const float dz = h * k.template slope<ACT>(e, v, d);
      s1[e] += dz;
      s2[e] = fmaf(dz, d, s2[e]);
    };
    int it = 0;
    for (; it + U <= me.full; it += U, p += U * hop, g += U * hop) {
      Pack<T, V> f[U], h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u].load(p + u * hop), h[u].load(g + u * hop);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[V], d[V];
        f[u].get(v);
        h[u].get(d);
#pragma unroll
        for (int e = 0; e < V; ++e) add(e, v[e], d[e]);
      }
    }
    for (; it < me.full; ++it, p += hop, g += hop) {
      Pack<T, V> f, h;
      f.load(p);
      h.load(g);
      float v[V], d[V];
      f.get(v);
      h.get(d);
#pragma unroll
      for (int e = 0; e < V; ++e) add(e, v[e], d[e]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (e < me.rest) add(e, Io<T>::to(p[e]), Io<T>::to(g[e]));
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
    o[1] = q * (float)stats[2 * (b * cut.G + c / cut.Cg) + 1];
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
  constexpr int V = Io<T>::V, U = 2;
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
  const long blk = (long)gridDim.x - 1 - blockIdx.x;      // in reverse order, as in the forward pass
  const long b = blk / cut.nchunk, ch = blk % cut.nchunk;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    const Share me = share_of<V>(cut, ch, t);
    if (me.full + me.rest == 0) continue;
    const T* p = x + b * cut.S + me.at;
    const T* g = dy + b * cut.S + me.at;
    T* o = dx + b * cut.S + me.at;
    const long hop = (long)cut.row * V;
    Channel<V> k;
    int c = (int)(((long)t * V) % cut.C);
    k.load(stats + 2 * b * cut.G, gamma, beta, c, cut.C, cut.Cg);
    float k1[V], k2[V];           // dx = a dz - k1 - (x - mean) k2
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const long bg = b * cut.G + c / cut.Cg;
      const float rstd = (float)stats[2 * bg + 1];
      k1[e] = coef[2 * bg] * rstd;
      k2[e] = coef[2 * bg + 1] * rstd * rstd;
      if (++c == cut.C) c = 0;
    }
    auto value = [&](int e, float v, float h) {
      float d;
      const float dz = h * k.template slope<ACT>(e, v, d);
      return fmaf(k.a[e], dz, -fmaf(d, k2[e], k1[e]));
    };
    int it = 0;
    for (; it + U <= me.full; it += U, p += U * hop, g += U * hop, o += U * hop) {
      Pack<T, V> f[U], h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u].load(p + u * hop), h[u].load(g + u * hop);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[V], d[V];
        f[u].get(v);
        h[u].get(d);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = value(e, v[e], d[e]);
        f[u].set(v);
        f[u].store(o + u * hop);
      }
    }
    for (; it < me.full; ++it, p += hop, g += hop, o += hop) {
      Pack<T, V> f, h;
      f.load(p);
      h.load(g);
      float v[V], d[V];
      f.get(v);
      h.get(d);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = value(e, v[e], d[e]);
      f.set(v);
      f.store(o);
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < me.rest) o[e] = Io<T>::from(value(e, Io<T>::to(p[e]), Io<T>::to(g[e])));
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
  // chunks: about four blocks of 256 threads for every compute unit over the whole batch, at least eight rows each (a
  // block's prologue and the joining of its sums cost about as much as four)
  long iters = (rows * batch + 1023) / 1024;
  if (iters < 8) iters = 8;
  if (iters > rows) iters = rows;
  cut->iters = (int)iters;
  cut->nchunk = (rows + iters - 1) / iters;
  const int threads = (cut->active + 63) / 64 * 64;
  cut->team = 64;
  while (cut->team > 1 && threads / cut->team < G) cut->team >>= 1;
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
