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
  static constexpr bool FINE = true;     // which of the activations below
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Io<bf16_t> {
  static constexpr int V = 8;
  static constexpr bool FINE = false;
  static __device__ __forceinline__ float to(bf16_t v) { return __uint_as_float((unsigned)v.b << 16); }
  static __device__ __forceinline__ bf16_t from(float v) { return bf16_t{f32_to_bf16(v)}; }
};
template <> struct Io<fp16_t> {
  static constexpr int V = 8;
  static constexpr bool FINE = false;
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
  __device__ __forceinline__ void load_once(const T* p) {
    raw = __builtin_nontemporal_load(reinterpret_cast<const decltype(raw)*>(p));
  }
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

// The activations, in two grades, both from the hardware's exponential and reciprocal (each good to about 1 unit of
// float32).  The kernels on 16-bit maps are bound by the vector unit as much as by memory, so theirs are written for few
// instructions.  For GELU
//   Phi(z) = 1 - e P(t) for z >= 0, e P(t) for z < 0,  e = exp(-z^2 / 2),  t = 1 / (1 + p |z| / sqrt 2),
// which shares its exponential with the density in the slope; t times a polynomial in t stands for the scaled
// erfcx(|z| / sqrt 2) / 2.  The coefficients come from a least-maximum fit over |z| < 13.4 in which an error of Phi of
// 1e-7 weighs as much as a relative one of 2e-5: 2e-8 of Phi near zero, 4e-6 relative in the tail (half a unit of fp16:
// 5e-4).
// FINE, for float32 maps: an exponential whose argument carries its rounding along, and Phi for |z| <= 1 as 1/2 + z Q(z^2),
// beyond as above from a fit of its own (relative error 6e-8, half a unit; Q: 1e-9).  Every value is within 4 units of its
// own size (GELU from -12 to -1) or 2 (elsewhere); memory still bounds the passes (8 x 65536 x 256 GELU: forward 307 us,
// 303 with the coarse grade; 32 x 2080 x 64: 14.7, 13.2).
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
// 2^(x (scale + scale_lo) + more), x * scale being rounded; 0 or infinity at either end
__device__ __forceinline__ float fine_exp2(float x, float scale, float scale_lo, float more) {
  const float h = x * scale, l = fmaf(x, scale, -h) + fmaf(x, scale_lo, more);
  return __builtin_amdgcn_exp2f(h) * fmaf(__builtin_amdgcn_fmed3f(l, -1.f, 1.f), 0.69314718055994531f, 1.f);
}
constexpr double LOG2_E = 1.44269504088896340736;
template <bool FINE>
__device__ __forceinline__ float sigmoid(float z) {
  const float e = FINE ? fine_exp2(z, (float)-LOG2_E, (float)((double)(float)LOG2_E - LOG2_E), 0.f) : fast_exp(-z);
  return __builtin_amdgcn_rcpf(1.f + e);
}
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  if (FINE) {
    constexpr float scale = (float)(-0.5 * LOG2_E);
    const float r = fminf(fabsf(z), 64.f), s = r * r;
    e = fine_exp2(s, scale, (float)(-0.5 * LOG2_E - (double)scale), fmaf(r, r, -s) * scale);
    float q = fmaf(s, -7.65420966e-06f, 0.000113486375f);
    q = fmaf(s, q, -0.00118632994f);
    q = fmaf(s, q, 0.00997332341f);
    q = fmaf(s, q, -0.0664903599f);
    q = fmaf(s, q, 0.39894228f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3938f * 0.70710678118654752f, fabsf(z), 1.f));
    float p = fmaf(t, 0.5f * -0.121039647f, 0.5f * 0.275834937f);
    p = fmaf(t, p, 0.5f * -0.0192640351f);
    p = fmaf(t, p, 0.5f * 0.226235426f);
    p = fmaf(t, p, 0.5f * 0.192260755f);
    p = fmaf(t, p, 0.5f * 0.22373901f);
    p = fmaf(t, p, 0.5f * 0.222097661f);
    p *= t * e;
    return fabsf(z) <= 1.f ? fmaf(z, q, 0.5f) : z < 0.f ? p : 1.f - p;
  }
  e = __builtin_amdgcn_exp2f(z * ((float)(-0.5 * LOG2_E) * z));
  const float t = __builtin_amdgcn_rcpf(fmaf(0.362f * 0.70710678118654752f, fabsf(z), 1.f));
  float p = fmaf(t, 0.5f * -0.158929867f, 0.5f * 0.534791676f);
  p = fmaf(t, p, 0.5f * -0.314430907f);
  p = fmaf(t, p, 0.5f * 0.399861424f);
  p = fmaf(t, p, 0.5f * 0.119611093f);
  p = fmaf(t, p, 0.5f * 0.215599491f);
  p = fmaf(t, p, 0.5f * 0.203497056f);
  p *= t * e;
  return z < 0.f ? p : 1.f - p;
}
template <int ACT, bool FINE>
__device__ __forceinline__ float act_fwd(float z) {
  if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
  if (ACT == ACT_SILU) return z * sigmoid<FINE>(z);
  if (ACT == ACT_GELU) {
    float e;
    return z * normal_cdf<FINE>(z, e);
  }
  return z;
}
template <int ACT, bool FINE>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == ACT_RELU) return z <= 0.f ? 0.f : 1.f;       // NaN stays NaN
  if (ACT == ACT_SILU) {
    const float s = sigmoid<FINE>(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == ACT_GELU) {
    float e;
    const float c = normal_cdf<FINE>(z, e);
    return fmaf(z * 0.39894228040143268f, e, c);
  }
  return 1.f;
}

// How a sample is cut: `active` threads of a block cover rows of `active` vectors (a multiple of the period), `columns`
// of them one after another where the period is longer than a block; a chunk is at most `iters` such rows.
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

// A thread's chain of 32-bit additions is a run of at most this many rows; the totals of a chunk's runs, at most as many,
// are a second chain.  One chain for a whole chunk would drift as maps grow: equal addends by 170 half units over 1024
// rows, by 10 over 64.
constexpr int GN_RUN = 64;

// sum over aligned teams of `team` lanes, the same in every lane of a team
__device__ __forceinline__ double team_sum(double v, int team) {
  for (int s = 1; s < team; s <<= 1) v += __shfl_xor(v, s);
  return v;
}

// A thread's share of a chunk: `full` whole vectors, `hop` values apart, from the first on; then possibly the sample's
// last, shorter one.  A chunk takes every nchunk-th row of threads, so that all blocks sweep through the sample together:
// blocks that each stream a run of their own, a power of two apart, crowd on a few memory channels.
struct Share {
  long at, hop;
  int full;
  int rest;     // values of the short vector behind them, 0: none
};
template <int V>
__device__ __forceinline__ Share share_of(const Cut& cut, long ch, int t) {
  const long v0 = ch * cut.row + t, step = cut.nchunk * cut.row, whole = cut.S / V;
  Share s;
  s.at = v0 * V;
  s.hop = step * V;
  const long n = v0 < whole ? (whole - v0 + step - 1) / step : 0;
  s.full = (int)n;
  s.rest = v0 + n * step == whole ? (int)(cut.S - whole * V) : 0;
  return s;
}

// ---------------------------------------------------------------------------------------------------- statistics
// Every thread sums d = x - k and d^2 per channel over a run of rows, k being the run's first value: as k is one of the
// n values summed, their sum of squares about it is at most n + 1 times that about their mean, so cancellation costs n
// roundings at most, whatever the mean of the map is -- hence runs of 64, however long the chunk.  Runs (in 32 bits),
// threads, chunks and channels (in 64) are joined by the parallel-variance formula
//   M2 = sum M2_i + sum n_i (mean_i - mean)^2.
// ONCE: the map is larger than what the last-level cache would keep for the next pass; reading it past that cache spares
// the eviction of dirty lines (268 MB: 49 us instead of 80, 5.5 TB/s; at 128 MB the two ways are within 5 %).
// Bound by memory: a map is read once here and once by the pass behind.  Four loads in flight per thread, four blocks of
// 256 threads a compute unit.  The joining afterwards took most of the time of a short chunk while a group's slots were
// added up one after another: hence teams of lanes per group, and one slot for a whole vector.
template <typename T, bool ONCE>
__global__ __launch_bounds__(1024) void gn_stats_kernel(const T* __restrict__ x, const Cut cut,
                                                        double* __restrict__ part) {
  constexpr int V = Io<T>::V, U = 4;            // U loads in flight per thread
  extern __shared__ float sh[];                 // [3][slots]: mean, M2, count of every slot
  const int tid = threadIdx.x;
  const long b = blockIdx.x / cut.nchunk, ch = blockIdx.x % cut.nchunk;
  const T* xs = x + b * cut.S;
  // a slot is a value of a thread's vectors, or all V of them where they belong to one group
  const bool whole = cut.Cg % V == 0;
  const int each = whole ? V : 1, C = cut.C / each, Cg = cut.Cg / each;
  const int slots = (cut.columns == 1 ? cut.active * V : cut.period * V) / each;
  float* smean = sh;
  float* sm2 = sh + slots;
  float* scnt = sh + 2 * slots;
  // a run's values are joined to those before it in their place
  auto leave = [&](int at, bool first, float n, float mean, float m2) {
    if (!first) {
      const float n0 = scnt[at], d = mean - smean[at], share = n / (n0 + n);
      m2 += fmaf(d * d, n0 * share, sm2[at]);
      mean = fmaf(d, share, smean[at]);
      n += n0;
    }
    smean[at] = mean;
    sm2[at] = m2;
    scnt[at] = n;
  };
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    const Share me = share_of<V>(cut, ch, t);
    const T* p = xs + me.at;
    const long hop = me.hop;
    int left = me.full;
    bool first = true;
    do {
      const int run = left < GN_RUN ? left : GN_RUN, rest = left == run ? me.rest : 0;
      left -= run;
      float k[V], s[V], q[V];
#pragma unroll
      for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
      if (run) {
        Pack<T, V> f;
        f.load(p);
        f.get(k);
      }
      int it = 0;
      for (; it + U <= run; it += U, p += U * hop) {
        Pack<T, V> f[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (ONCE)
            f[u].load_once(p + u * hop);
          else
            f[u].load(p + u * hop);
        }
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
      for (; it < run; ++it, p += hop) {
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
      float n[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (e < rest) {
          const float v = Io<T>::to(p[e]);
          if (!run) k[e] = v;
          const float d = v - k[e];
          s[e] += d;
          q[e] = fmaf(d, d, q[e]);
        }
        n[e] = (float)(run + (e < rest ? 1 : 0));
        const float m = n[e] > 0.f ? s[e] / n[e] : 0.f;
        q[e] = fmaxf(fmaf(-s[e], m, q[e]), 0.f);
        s[e] = m;                                 // now the mean and M2 about it, k being the origin
      }
      if (whole) {                                // (a short vector leaves whole groups' values out at its end)
        float count = 0.f, sum = 0.f, m2 = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[e] += k[e] - k[0];
          count += n[e];
          sum = fmaf(n[e], s[e], sum);
        }
        const float m = count > 0.f ? sum / count : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = s[e] - m;
          m2 += n[e] > 0.f ? fmaf(n[e] * d, d, q[e]) : 0.f;
        }
        leave(t, first, count, k[0] + m, m2);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) leave(t * V + e, first, n[e], k[e] + s[e], q[e]);
      }
      first = false;
    } while (left > 0);
  }
  __syncthreads();
  // a team of lanes per group, all groups at once where there are enough threads; slot q belongs to channel
  // (or V channels) q % C (slots is a multiple of C)
  const int per = slots / C * Cg;
  const int lane = tid & (cut.team - 1), teams = blockDim.x / cut.team;
  for (int g0 = 0; g0 < cut.G; g0 += teams) {          // uniform: all lanes take part in the sums
    const int g = g0 + tid / cut.team;
    const bool mine = g < cut.G;
    double n = 0.0, sum = 0.0;
    for (int i = lane; mine && i < per; i += cut.team) {
      const int q = (i / Cg) * C + g * Cg + i % Cg;
      n += (double)scnt[q];
      sum += (double)scnt[q] * (double)smean[q];
    }
    n = team_sum(n, cut.team);
    sum = team_sum(sum, cut.team);
    const double mean = n > 0.0 ? sum / n : 0.0;
    double m2 = 0.0;
    for (int i = lane; mine && i < per; i += cut.team) {
      const int q = (i / Cg) * C + g * Cg + i % Cg;
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
// y = act((x - mean) a + beta), a = gamma rstd.  Bound by memory: 8 x 65536 x 256 bf16 with SiLU 94 us, 537 MB at
// 5.7 TB/s.  Blocks and threads go through the map in the opposite order of the statistics pass, so that what that pass
// read last is taken from the last-level cache (4 x 16384 x 512 bf16: 29 us, behind statistics of 25 us).
template <typename T, int ACT, bool ONCE>
__global__ __launch_bounds__(1024) void gn_apply_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                        const float* __restrict__ beta,
                                                        const double* __restrict__ stats, T* __restrict__ y,
                                                        const Cut cut) {
  constexpr int V = Io<T>::V, U = 4;
  const int tid = threadIdx.x;
  const long blk = (long)gridDim.x - 1 - blockIdx.x, b = blk / cut.nchunk, ch = blk % cut.nchunk;   // reversed too
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    const Share me = share_of<V>(cut, ch, t);
    if (me.full + me.rest == 0) continue;
    const T* p = x + b * cut.S + me.at;
    T* o = y + b * cut.S + me.at;
    const long hop = me.hop;
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
    // backwards: what the statistics pass read last is still in the cache
    p += me.full * hop;
    o += me.full * hop;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < me.rest) o[e] = Io<T>::from(act_fwd<ACT, Io<T>::FINE>(fmaf(Io<T>::to(p[e]) - mean[e], a[e], c0[e])));
    auto map = [&](Pack<T, V>& f) {
      float v[V];
      f.get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = act_fwd<ACT, Io<T>::FINE>(fmaf(v[e] - mean[e], a[e], c0[e]));
      f.set(v);
    };
    int it = me.full;
    for (; it >= U; it -= U) {
      p -= U * hop;
      o -= U * hop;
      Pack<T, V> f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (ONCE)
          f[u].load_once(p + u * hop);
        else
          f[u].load(p + u * hop);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        map(f[u]);
        f[u].store(o + u * hop);
      }
    }
    for (; it > 0; --it) {
      p -= hop;
      o -= hop;
      Pack<T, V> f;
      f.load(p);
      map(f);
      f.store(o);
    }
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
  template <int ACT, bool FINE>
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
    return act_slope<ACT, FINE>(z);
  }
  // dz of one value; behind a ReLU the gradient is selected, so that no infinity or NaN of dy gets past a closed one
  template <int ACT, bool FINE>
  __device__ __forceinline__ float grad(int e, float x, float dy, float& d) const {
    const float s = slope<ACT, FINE>(e, x, d);
    return ACT == ACT_RELU ? (s != 0.f ? dy : 0.f) : dy * s;
  }
};

// Per chunk and channel: sum of dz and of dz xhat (rstd is one factor, applied at the end).  A thread sums runs of at most
// 64 rows in 32 bits and adds them up in its place in LDS; threads and chunks are joined in 64 bits, their sums kept in
// 32 in between.  4 x 16384 x 512 bf16, SiLU: 31 us, 134 MB at 4.3 TB/s; the vector unit is as busy as memory (the slope
// of an activation is 12 to 20 instructions a value).
// RUNS: chunks of more than one run; such maps are read past the cache anyway, and the others keep the registers.
template <typename T, int ACT, bool ONCE, bool RUNS>
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
    const long hop = me.hop;
    Channel<V> k;
    k.load(stats + 2 * b * cut.G, gamma, beta, (int)(((long)t * V) % cut.C), cut.C, cut.Cg);
    float s1[V], s2[V];           // sums of dz and of dz (x - mean)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s1[e] = s2[e] = 0.f;
      if (RUNS) sh[t * V + e] = sh[slots + t * V + e] = 0.f;
    }
    auto add = [&](int e, float v, float h) {
      float d;
      const float dz = k.template grad<ACT, Io<T>::FINE>(e, v, h, d);
      s1[e] += dz;
      s2[e] = fmaf(dz, d, s2[e]);
    };
    // a run's sums are added to those before it in the thread's place in LDS
    auto leave = [&]() {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sh[t * V + e] = RUNS ? sh[t * V + e] + s1[e] : s1[e];
        sh[slots + t * V + e] = RUNS ? sh[slots + t * V + e] + s2[e] : s2[e];
        s1[e] = s2[e] = 0.f;
      }
    };
    int it = 0;
    for (; it + U <= me.full; it += U, p += U * hop, g += U * hop) {
      if (RUNS && it && it % GN_RUN == 0) leave();
      Pack<T, V> f[U], h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (ONCE)
          f[u].load_once(p + u * hop), h[u].load_once(g + u * hop);
        else
          f[u].load(p + u * hop), h[u].load(g + u * hop);
      }
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
    for (int e = 0; e < V; ++e)
      if (e < me.rest) add(e, Io<T>::to(p[e]), Io<T>::to(g[e]));
    leave();
  }
  __syncthreads();
  for (int c = tid; c < cut.C; c += blockDim.x) {
    double a = 0.0, q = 0.0;
    for (int r = c; r < slots; r += cut.C) {
      a += (double)sh[r];
      q += (double)sh[slots + r];
    }
    float* o = part + ((long)blockIdx.x * cut.C + c) * 2;
    o[0] = (float)a;
    o[1] = (float)(q * stats[2 * (b * cut.G + c / cut.Cg) + 1]);
  }
}

// Joins the chunks: channel sums [b][c][2].  A block has up to 64 channels of a sample, a channel per lane, the chunks
// shared out among its waves and joined in order.  Where a block's channels are whole groups (`span` = 64 / Cg * Cg) it
// also leaves the two means of each over N values; larger groups are joined by the kernel behind this one.
__global__ __launch_bounds__(1024) void gn_bwd_join_kernel(const float* __restrict__ part, const Cut cut, int span,
                                                           const float* __restrict__ gamma, float* __restrict__ sums,
                                                           float* __restrict__ coef) {
  __shared__ double red[16][64][2];
  const int blocks = (cut.C + span - 1) / span;
  const long b = blockIdx.x / blocks;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int c0 = blockIdx.x % blocks * span, c = c0 + lane;
  const bool mine = lane < span && c < cut.C;
  double a = 0.0, q = 0.0;
  if (mine) {
    const float* p = part + (b * cut.nchunk * cut.C + c) * 2;
#pragma unroll 4
    for (long i = w; i < cut.nchunk; i += nw) {
      a += (double)p[i * cut.C * 2];
      q += (double)p[i * cut.C * 2 + 1];
    }
  }
  red[w][lane][0] = a;
  red[w][lane][1] = q;
  __syncthreads();
  if (w) return;
  for (int k = 1; k < nw; ++k) {
    a += red[k][lane][0];
    q += red[k][lane][1];
  }
  if (mine) {
    sums[(b * cut.C + c) * 2] = (float)a;
    sums[(b * cut.C + c) * 2 + 1] = (float)q;
  }
  if (cut.Cg > 64) return;
  const double gm = mine && gamma ? (double)gamma[c] : 1.0;
  red[0][lane][0] = a * gm;
  red[0][lane][1] = q * gm;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (lane < span / cut.Cg && c0 + lane * cut.Cg < cut.C) {
    double c1 = 0.0, c2 = 0.0;
    for (int i = lane * cut.Cg; i < (lane + 1) * cut.Cg; ++i) {
      c1 += red[0][i][0];
      c2 += red[0][i][1];
    }
    const double n = (double)(cut.S / cut.C) * cut.Cg;
    float* o = coef + 2 * (b * cut.G + c0 / cut.Cg + lane);
    o[0] = (float)(c1 / n);
    o[1] = (float)(c2 / n);
  }
}

// the two means of a group of more than 64 channels from their sums
__global__ __launch_bounds__(256) void gn_bwd_coef_kernel(const float* __restrict__ sums, const Cut cut,
                                                          const float* __restrict__ gamma, float* __restrict__ coef) {
  __shared__ double red[16];
  const long b = blockIdx.x / cut.G;
  const int c0 = blockIdx.x % cut.G * cut.Cg;
  double c1 = 0.0, c2 = 0.0;
  for (int c = c0 + threadIdx.x; c < c0 + cut.Cg; c += 256) {
    const double gm = gamma ? (double)gamma[c] : 1.0;
    c1 += (double)sums[(b * cut.C + c) * 2] * gm;
    c2 += (double)sums[(b * cut.C + c) * 2 + 1] * gm;
  }
  c1 = block_sum_d(c1, red);
  c2 = block_sum_d(c2, red);
  if (threadIdx.x == 0) {
    const double n = (double)(cut.S / cut.C) * cut.Cg;
    coef[2 * blockIdx.x] = (float)(c1 / n);
    coef[2 * blockIdx.x + 1] = (float)(c2 / n);
  }
}

// dgamma / dbeta of 64 channels: a channel per lane, the samples shared out among the block's waves, joined in order
__device__ __forceinline__ void param_sums(const float* __restrict__ sums, long batch, int C, int c0,
                                           float* __restrict__ dgamma, float* __restrict__ dbeta, double (*red)[64][2]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, c = c0 + lane;
  double a = 0.0, q = 0.0;
  if (c < C) {
#pragma unroll 4
    for (long b = w; b < batch; b += nw) {
      a += (double)sums[(b * C + c) * 2];
      q += (double)sums[(b * C + c) * 2 + 1];
    }
  }
  red[w][lane][0] = a;
  red[w][lane][1] = q;
  __syncthreads();
  if (w || c >= C) return;
  for (int k = 1; k < nw; ++k) {
    a += red[k][lane][0];
    q += red[k][lane][1];
  }
  if (dbeta) dbeta[c] = (float)a;
  if (dgamma) dgamma[c] = (float)q;
}
__global__ __launch_bounds__(1024) void gn_param_kernel(const float* __restrict__ sums, long batch, int C,
                                                        float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ double red[16][64][2];
  param_sums(sums, batch, C, blockIdx.x * 64, dgamma, dbeta, red);
}

// Blocks [0, nparam): dgamma / dbeta; the others: dx = a dz - k1 - (x - mean) k2 from x and dy read again, dz formed again
// (storing it would cost a write and a read of the map).  4 x 16384 x 512 bf16, SiLU: 41 us, 201 MB at 4.9 TB/s.
template <typename T, int ACT, bool ONCE>
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
    __shared__ double red[16][64][2];
    param_sums(sums, batch, cut.C, blockIdx.x * 64, dgamma, dbeta, red);
    return;
  }
  const long blk = (long)gridDim.x - 1 - blockIdx.x;      // the samples in reverse order too
  const long b = blk / cut.nchunk, ch = blk % cut.nchunk;
  for (int col = 0; col < cut.columns; ++col) {
    const int t = col * cut.active + tid;
    if (tid >= cut.active || t >= cut.row) continue;
    const Share me = share_of<V>(cut, ch, t);
    if (me.full + me.rest == 0) continue;
    const T* p = x + b * cut.S + me.at;
    const T* g = dy + b * cut.S + me.at;
    T* o = dx + b * cut.S + me.at;
    const long hop = me.hop;
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
      const float dz = k.template grad<ACT, Io<T>::FINE>(e, v, h, d);
      return fmaf(k.a[e], dz, -fmaf(d, k2[e], k1[e]));
    };
    p += me.full * hop;           // backwards, as in the forward pass
    g += me.full * hop;
    o += me.full * hop;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < me.rest) o[e] = Io<T>::from(value(e, Io<T>::to(p[e]), Io<T>::to(g[e])));
    int it = me.full;
    for (; it >= U; it -= U) {
      p -= U * hop;
      g -= U * hop;
      o -= U * hop;
      Pack<T, V> f[U], h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (ONCE)
          f[u].load_once(p + u * hop), h[u].load_once(g + u * hop);
        else
          f[u].load(p + u * hop), h[u].load(g + u * hop);
      }
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
    for (; it > 0; --it) {
      p -= hop;
      g -= hop;
      o -= hop;
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
  }
}

// ------------------------------------------------------------------------------------- groups that fit one block
// A block keeps its slab -- the P positions of `bundle` groups of one sample -- in registers: one read, one launch, no
// partial sums.  Thread t always has the same W channels (column t % nw of a row of the slab) and every rp-th row.  The
// statistics take two passes over the registers, the second one correcting the mean of the first:
//   m = sum x / N,  d = x - m,  mean = m + sum d / N,  var = (sum d^2 - (sum d)^2 / N) / N,
// exact to rounding whatever the mean is.  A bundle has at least 64 bytes of a row where enough blocks remain; the
// bundles of one sample run on one XCD, whose L2 they share.
// One launch instead of three, one read instead of two.  256 x 512 x 128 bf16 in 16 groups, SiLU: 21 us, 67 MB at 3.2 TB/s
// (chunks: 40 us); 32 x 2080 x 64 fp32 in 8 groups, ReLU: 15 us (22), backward 18.6 + 3.8 us (28); 1 x 128 x 256 in 32
// groups: 4.7 us, which is the launch and two joins.  Bound by the wait for a block's own loads: its two sums cannot
// start before.
struct Slab {
  long S;          // values per sample
  int P, C, G, Cg;
  int W;           // values per vector, divides Cg
  int bundle;      // groups per block
  int bundles;     // blocks per sample
  int nw, rp;      // vectors in a row of the slab, rows per pass of the block
  int threads, vecs;
  long batch;
};
struct Place {
  long b;
  int c0, L, nw, G;     // first channel, channels, vectors a row, groups
};
__device__ __forceinline__ Place place_of(const Slab& q) {
  // eight samples side by side, one per XCD
  const long l = blockIdx.x, per = 8l * q.bundles, eights = q.batch >> 3;
  Place p;
  long k;
  if (l < eights * per) {
    p.b = l / per * 8 + (l & 7);
    k = l % per >> 3;
  } else {
    const long r = l - eights * per;
    p.b = eights * 8 + r / q.bundles;
    k = r % q.bundles;
  }
  const int g0 = (int)k * q.bundle;
  p.G = q.G - g0 < q.bundle ? q.G - g0 : q.bundle;
  p.c0 = g0 * q.Cg;
  p.L = p.G * q.Cg;
  p.nw = p.L / q.W;
  return p;
}

// sums over the groups of two values per thread; `out` holds them for every group afterwards
__device__ __forceinline__ void group_sums(float a, float b, const Slab& q, const Place& p, float2* red,
                                           double (*out)[2]) {
  const int tid = threadIdx.x, cw = q.Cg / q.W, per = q.rp * cw;
  if (p.G == 1) {                               // uniform: the whole block is one group
    const double s = wave_sum_d((double)a), t = wave_sum_d((double)b);
    double2* part = reinterpret_cast<double2*>(red);
    __syncthreads();
    if ((tid & 63) == 0) part[tid >> 6] = make_double2(s, t);
    __syncthreads();
    double2 all = make_double2(0.0, 0.0);
    for (int k = 0; k < (int)blockDim.x >> 6; ++k) all.x += part[k].x, all.y += part[k].y;
    if (tid == 0) out[0][0] = all.x, out[0][1] = all.y;
    __syncthreads();
    return;
  }
  __syncthreads();
  red[tid] = make_float2(a, b);
  __syncthreads();
  int team = 64;
  while (team > 1 && (int)blockDim.x / team < p.G) team >>= 1;
  const int lane = tid & (team - 1), teams = blockDim.x / team;
  for (int g0 = 0; g0 < p.G; g0 += teams) {
    const int g = g0 + tid / team;
    double s = 0.0, t = 0.0;
    for (int i = lane; g < p.G && i < per; i += team) {
      const float2 v = red[(i / cw) * q.nw + g * cw + i % cw];
      s += (double)v.x;
      t += (double)v.y;
    }
    s = team_sum(s, team);
    t = team_sum(t, team);
    if (g < p.G && lane == 0) {
      out[g][0] = s;
      out[g][1] = t;
    }
  }
  __syncthreads();
}

template <typename T, int W, int NV, int ACT>
__device__ __forceinline__ void slab_store(Pack<T, W> (&f)[NV], const float (&mean)[W], const float (&a)[W],
                                           const float (&bet)[W], T* y, int r0, const Slab& q) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int r = r0 + k * q.rp;
    if (r < q.P) {
      float v[W];
      f[k].get(v);
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = act_fwd<ACT, Io<T>::FINE>(fmaf(v[e] - mean[e], a[e], bet[e]));
      f[k].set(v);
      f[k].store(y + (long)r * q.C);
    }
  }
}

constexpr int GN_MAX_BUNDLE = 64;

template <typename T, int W, int NV>
__global__ __launch_bounds__(1024) void gn_slab_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, T* __restrict__ y,
                                                           double* __restrict__ stats, float eps, int act,
                                                           const Slab q) {
  __shared__ __attribute__((aligned(16))) float2 red[1024];      // read as double2 too
  __shared__ double sum[GN_MAX_BUNDLE][2];
  const Place p = place_of(q);
  const int tid = threadIdx.x, col = tid % q.nw, r0 = tid / q.nw;
  const bool in = col < p.nw && r0 < q.rp;
  const long at = p.b * q.S + p.c0 + col * W;
  Pack<T, W> f[NV];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int r = r0 + k * q.rp;
    if (in && r < q.P) f[k].load(x + at + (long)r * q.C);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (in && r0 + k * q.rp < q.P) {
      float v[W];
      f[k].get(v);
#pragma unroll
      for (int e = 0; e < W; ++e) s += v[e];
    }
  }
  float gam[W], bet[W];                         // asked for now, needed at the end
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const int c = in ? p.c0 + col * W + e : 0;
    gam[e] = gamma ? gamma[c] : 1.f;
    bet[e] = beta ? beta[c] : 0.f;
  }
  const int g = in ? col * W / q.Cg : 0;
  const double n = (double)q.P * q.Cg;
  group_sums(s, 0.f, q, p, red, sum);
  const double m0 = sum[g][0] / n;
  const float m = (float)m0;
  float d1 = 0.f, d2 = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (in && r0 + k * q.rp < q.P) {
      float v[W];
      f[k].get(v);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float d = v[e] - m;
        d1 += d;
        d2 = fmaf(d, d, d2);
      }
    }
  }
  group_sums(d1, d2, q, p, red, sum);
  const double off = sum[g][0] / n;
  const double var = fmax(sum[g][1] / n - off * off, 0.0);
  const double mean64 = (double)m + off;
  // a NaN of the data passes fmax by: put it back
  const double rstd64 = sum[g][1] == sum[g][1] ? 1.0 / sqrt(var + (double)eps) : sum[g][1];
  if (stats && in && r0 == 0 && col * W % q.Cg == 0) {
    double* o = stats + 2 * (p.b * q.G + p.c0 / q.Cg + g);
    o[0] = mean64;
    o[1] = rstd64;
  }
  if (!in) return;
  float mean[W], a[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    mean[e] = (float)mean64;
    a[e] = (float)rstd64 * gam[e];
  }
  T* o = y + at;
  switch (act) {
    case ACT_NONE: slab_store<T, W, NV, ACT_NONE>(f, mean, a, bet, o, r0, q); break;
    case ACT_RELU: slab_store<T, W, NV, ACT_RELU>(f, mean, a, bet, o, r0, q); break;
    case ACT_SILU: slab_store<T, W, NV, ACT_SILU>(f, mean, a, bet, o, r0, q); break;
    default: slab_store<T, W, NV, ACT_GELU>(f, mean, a, bet, o, r0, q); break;
  }
}

// The backward pass of a slab: dx, and the sums of its channels for the parameter gradients.
template <typename T, int W, int NV, int ACT>
__global__ __launch_bounds__(1024) void gn_slab_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                           const float* __restrict__ gamma,
                                                           const float* __restrict__ beta,
                                                           const double* __restrict__ stats, T* __restrict__ dx,
                                                           float* __restrict__ sums, const Slab q) {
  extern __shared__ float sh[];                 // [rows][channels][2], then [segments][channels][2]
  __shared__ double sum[GN_MAX_BUNDLE][2];
  const Place p = place_of(q);
  const int tid = threadIdx.x, col = tid % q.nw, r0 = tid / q.nw;
  const bool in = col < p.nw && r0 < q.rp;
  const long at = p.b * q.S + p.c0 + col * W;
  const double* st = stats + 2 * p.b * q.G;
  Pack<T, W> f[NV], h[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int r = r0 + k * q.rp;
    if (in && r < q.P) {
      f[k].load(x + at + (long)r * q.C);
      h[k].load(dy + at + (long)r * q.C);
    }
  }
  Channel<W> ch;
  ch.load(st, gamma, beta, in ? p.c0 + col * W : p.c0, q.C, q.Cg);
  float s1[W], s2[W];
#pragma unroll
  for (int e = 0; e < W; ++e) s1[e] = s2[e] = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (in && r0 + k * q.rp < q.P) {
      float v[W], g[W];
      f[k].get(v);
      h[k].get(g);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        float d;
        const float dz = ch.template grad<ACT, Io<T>::FINE>(e, v[e], g[e], d);
        s1[e] += dz;
        s2[e] = fmaf(dz, d, s2[e]);
      }
    }
  }
  const int Lf = q.nw * W;                      // channels of a full bundle: the row pitch
  float* seg = sh + 2 * q.rp * Lf;
  if (r0 < q.rp) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      sh[(r0 * Lf + col * W + e) * 2] = s1[e];
      sh[(r0 * Lf + col * W + e) * 2 + 1] = s2[e];
    }
  }
  __syncthreads();
  // two stages of at most 32 additions one after another: more segments would leave their sum to a few threads
  const int spare = (int)blockDim.x / p.L, nseg = spare > 32 ? 32 : spare > 1 ? spare : 1;
  for (int i = tid; i < p.L * nseg; i += blockDim.x) {
    const int c = i % p.L;
    float a = 0.f, t = 0.f;
#pragma unroll 4
    for (int r = i / p.L; r < q.rp; r += nseg) {
      a += sh[(r * Lf + c) * 2];
      t += sh[(r * Lf + c) * 2 + 1];
    }
    seg[2 * i] = a;
    seg[2 * i + 1] = t;
  }
  __syncthreads();
  for (int c = tid; c < p.L; c += blockDim.x) {
    float a = 0.f, t = 0.f;
#pragma unroll 4
    for (int i = c; i < p.L * nseg; i += p.L) {
      a += seg[2 * i];
      t += seg[2 * i + 1];
    }
    t *= (float)st[2 * ((p.c0 + c) / q.Cg) + 1];
    float* o = sums + (p.b * q.C + p.c0 + c) * 2;
    o[0] = a;
    o[1] = t;
    const float gm = gamma ? gamma[p.c0 + c] : 1.f;
    sh[2 * c] = a * gm;
    sh[2 * c + 1] = t * gm;
  }
  if (!dx) return;
  __syncthreads();
  int team = 64;
  while (team > 1 && (int)blockDim.x / team < p.G) team >>= 1;
  const int lane = tid & (team - 1), teams = blockDim.x / team;
  for (int g0 = 0; g0 < p.G; g0 += teams) {
    const int g = g0 + tid / team;
    double a = 0.0, t = 0.0;
    for (int i = lane; g < p.G && i < q.Cg; i += team) {
      a += (double)sh[2 * (g * q.Cg + i)];
      t += (double)sh[2 * (g * q.Cg + i) + 1];
    }
    a = team_sum(a, team);
    t = team_sum(t, team);
    if (g < p.G && lane == 0) {
      sum[g][0] = a;
      sum[g][1] = t;
    }
  }
  __syncthreads();
  if (!in) return;
  const int g = col * W / q.Cg;
  const double n = (double)q.P * q.Cg;
  const float rstd = (float)st[2 * (p.c0 / q.Cg + g) + 1];
  const float k1 = (float)(sum[g][0] / n) * rstd, k2 = (float)(sum[g][1] / n) * rstd * rstd;
  T* o = dx + at;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int r = r0 + k * q.rp;
    if (r < q.P) {
      float v[W], gr[W];
      f[k].get(v);
      h[k].get(gr);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        float d;
        const float dz = ch.template grad<ACT, Io<T>::FINE>(e, v[e], gr[e], d);
        v[e] = fmaf(ch.a[e], dz, -fmaf(d, k2, k1));
      }
      f[k].set(v);
      f[k].store(o + (long)r * q.C);
    }
  }
}

// ---------------------------------------------------------------------------------------------------- host side
constexpr int GN_MAX_CHANNELS = 4096;
constexpr int GN_MAX_SLOTS = 12288;         // three floats of LDS for each: 144 of the 160 KiB
constexpr long GN_MAX_BLOCKS = 4000000;     // a grid's threads are counted in 32 bits, blocks have up to 1024
constexpr long GN_CACHED = 160l << 20;      // what a second pass still finds of the first one's reads in the 256 MB cache

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
  // of wide maps at least 32 positions as long as that leaves a block for every compute unit: a chunk's sums are two
  // floats a channel, written and read again
  const long deep = 32l * C / ((long)V * cut->row);
  if (iters < deep) iters = deep < rows * batch / 256 ? deep : iters > rows * batch / 256 ? iters : rows * batch / 256;
  if (iters > GN_RUN * GN_RUN) iters = GN_RUN * GN_RUN;
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
template <auto kernel>
int allow_lds(size_t bytes) {
  static PerDeviceOnce once;
  if (bytes > 65536 && once.pending()) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                            12 * GN_MAX_SLOTS) != hipSuccess)
      return MMSA_ERR_LAUNCH;
    once.done();
  }
  return MMSA_OK;
}

// What a pass costs in microseconds either way, from measurements over 1 to 64 samples of 256 to 8192 positions of 61 to
// 512 channels.  In registers: a block walks its P rows of `row` bytes at a pace of its own, and beyond 256 blocks they
// wait for each other; narrow rows cost nearly what wide ones do (64 samples of 8192 positions in 32 groups of 2 bf16
// channels: 176 us against 50 cut in chunks, backward 264 against 72; 16 samples of 4096 in groups of 16: 38 against 55).
// In chunks: the launches, and the bytes of all passes.
float slab_cost(const Slab& q, int dtype, bool backward) {
  const int size = dtype == 0 ? 4 : 2, row = q.bundle * q.Cg * size;
  const float blocks = (float)q.batch * q.bundles / 256.f, rounds = blocks > 1.f ? blocks : 1.f;
  return backward ? 10.f + 1e-3f * q.P * rounds * (3.f + (size == 4 ? .14f : .2f) * row)
                  : 6.f + 1e-3f * q.P * rounds * (2.4f + (size == 4 ? .05f : .0875f) * row);
}
float cut_cost(const Slab& q, int dtype, bool backward) {
  const float mb = 1e-6f * q.batch * q.S * (dtype == 0 ? 4 : 2);
  return backward ? (dtype == 0 ? 17.f + .75f * mb : 21.f + .8f * mb) : (dtype == 0 ? 14.f + .45f * mb : 18.f + .52f * mb);
}

// Whether a pass keeps its slabs in registers, and how.  `most`: registers of 4 bytes a thread may hold of one map.
bool make_slab(long batch, long positions, int C, int G, int dtype, int most, bool backward, Slab* q) {
  const int size = dtype == 0 ? 4 : 2, Cg = C / G;
  if (positions > 65536) return false;
  q->S = positions * C;
  q->P = (int)positions;
  q->C = C;
  q->G = G;
  q->Cg = Cg;
  q->batch = batch;
  q->W = 1;
  for (int w = 16 / size; w > 1; w >>= 1)
    if (Cg % w == 0 && (w == 16 / size || size * w == 8)) {
      q->W = w;
      break;
    }
  const int reg = (q->W * size + 3) / 4;        // registers of a vector
  int bundle = (64 + Cg * size - 1) / (Cg * size);
  if (bundle > G) bundle = G;
  if (batch * ((G + bundle - 1) / bundle) < 256) bundle = 1;
  for (; bundle >= 1; bundle >>= 1) {
    q->bundle = bundle;
    q->bundles = (G + bundle - 1) / bundle;
    q->nw = bundle * Cg / q->W;
    for (int t = 256; t <= 1024; t <<= 1) {
      if (q->nw > t) continue;
      q->rp = t / q->nw;
      q->threads = t;
      q->vecs = (q->P + q->rp - 1) / q->rp;
      const int cap = t < 1024 ? 4 : most / reg < 16 ? most / reg : 16;
      if (q->vecs <= cap)
        return batch * q->bundles <= GN_MAX_BLOCKS && slab_cost(*q, dtype, backward) <= cut_cost(*q, dtype, backward);
    }
  }
  return false;
}

template <typename T, int W, int NV>
int slab_fwd(const void* x, const float* gamma, const float* beta, void* y, double* stats, float eps, int act,
             const Slab& q, hipStream_t s) {
  hipLaunchKernelGGL((gn_slab_fwd_kernel<T, W, NV>), dim3((unsigned)(q.batch * q.bundles)), dim3(q.threads), 0, s,
                     static_cast<const T*>(x), gamma, beta, static_cast<T*>(y), stats, eps, act, q);
  return mmsa_launch_status();
}
template <typename T, int W>
int slab_fwd_n(const void* x, const float* gamma, const float* beta, void* y, double* stats, float eps, int act,
               const Slab& q, hipStream_t s) {
  if (q.vecs <= 4) return slab_fwd<T, W, 4>(x, gamma, beta, y, stats, eps, act, q, s);
  if (q.vecs <= 8) return slab_fwd<T, W, 8>(x, gamma, beta, y, stats, eps, act, q, s);
  return slab_fwd<T, W, 16>(x, gamma, beta, y, stats, eps, act, q, s);
}
size_t slab_lds(const Slab& q) {
  const size_t row = (size_t)q.nw * q.W, segs = row > (size_t)q.threads ? row : q.threads;
  return 8 * (q.rp * row + segs);
}
template <typename T, int W, int NV, int ACT>
int slab_bwd(const void* dy, const void* x, const float* gamma, const float* beta, const double* stats, void* dx,
             float* dgamma, float* dbeta, float* sums, const Slab& q, hipStream_t s) {
  const size_t lds = slab_lds(q);
  if (int rc = allow_lds<gn_slab_bwd_kernel<T, W, NV, ACT>>(lds)) return rc;
  hipLaunchKernelGGL((gn_slab_bwd_kernel<T, W, NV, ACT>), dim3((unsigned)(q.batch * q.bundles)), dim3(q.threads), lds, s,
                     static_cast<const T*>(dy), static_cast<const T*>(x), gamma, beta, stats, static_cast<T*>(dx), sums,
                     q);
  if (dgamma || dbeta)
    hipLaunchKernelGGL(gn_param_kernel, dim3((q.C + 63) / 64), dim3(1024), 0, s, sums, q.batch, q.C, dgamma, dbeta);
  return mmsa_launch_status();
}
template <typename T, int W, int ACT>
int slab_bwd_n(const void* dy, const void* x, const float* gamma, const float* beta, const double* stats, void* dx,
               float* dgamma, float* dbeta, float* sums, const Slab& q, hipStream_t s) {
  if (q.vecs <= 4) return slab_bwd<T, W, 4, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, sums, q, s);
  if constexpr (W * sizeof(T) < 16)
    return slab_bwd<T, W, 16, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, sums, q, s);
  else
    return slab_bwd<T, W, 6, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, sums, q, s);
}

// registers a thread may hold of one map: forward 64 of its 128; backward, which holds two maps and the channels'
// coefficients, 24 in 16-byte vectors, else 16 vectors
constexpr int FWD_REGS = 64, BWD_REGS = 24;

// the three launches of a map whose groups do not fit one block
template <typename T, bool ONCE>
int cut_fwd(const T* x, const float* gamma, const float* beta, T* y, double* stats, double* part, long batch,
            const Cut& cut, int dtype, float eps, int act, hipStream_t s) {
  const dim3 grid((unsigned)(batch * cut.nchunk)), block(block_of(cut));
  const size_t lds = 3 * sizeof(float) * slots_of(cut, dtype);
  if (int rc = allow_lds<gn_stats_kernel<T, ONCE>>(lds)) return rc;
  hipLaunchKernelGGL((gn_stats_kernel<T, ONCE>), grid, block, lds, s, x, cut, part);
  hipLaunchKernelGGL(gn_stats_join_kernel, dim3((unsigned)(batch * cut.G)), dim3(64), 0, s, (const double*)part,
                     cut.nchunk, cut.G, eps, stats);
#define GN_APPLY(A) \
  hipLaunchKernelGGL((gn_apply_kernel<T, A, ONCE>), grid, block, 0, s, x, gamma, beta, stats, y, cut)
  switch (act) {
    case ACT_NONE: GN_APPLY(ACT_NONE); break;
    case ACT_RELU: GN_APPLY(ACT_RELU); break;
    case ACT_SILU: GN_APPLY(ACT_SILU); break;
    default: GN_APPLY(ACT_GELU); break;
  }
#undef GN_APPLY
  return mmsa_launch_status();
}

template <typename T>
int gn_fwd(const void* x, const float* gamma, const float* beta, void* y, double* stats, void* scratch, long batch,
           const Cut& cut, int dtype, float eps, int act, hipStream_t s) {
  Slab q;
  if (make_slab(batch, cut.S / cut.C, cut.C, cut.G, dtype, FWD_REGS, false, &q)) {
    if (q.W == Io<T>::V) return slab_fwd_n<T, Io<T>::V>(x, gamma, beta, y, stats, eps, act, q, s);
    if constexpr (sizeof(T) == 2)
      if (q.W == 4) return slab_fwd_n<T, 4>(x, gamma, beta, y, stats, eps, act, q, s);
    if constexpr (sizeof(T) == 4)
      if (q.W == 2) return slab_fwd_n<T, 2>(x, gamma, beta, y, stats, eps, act, q, s);
    return slab_fwd_n<T, 1>(x, gamma, beta, y, stats, eps, act, q, s);
  }
  const T* xp = static_cast<const T*>(x);
  T* yp = static_cast<T*>(y);
  double* part = static_cast<double*>(scratch);
  MMSA_REQUIRE(scratch);
  if (!stats) stats = part + batch * cut.nchunk * cut.G * 3;
  if (batch * cut.S * (long)sizeof(T) > GN_CACHED)
    return cut_fwd<T, true>(xp, gamma, beta, yp, stats, part, batch, cut, dtype, eps, act, s);
  return cut_fwd<T, false>(xp, gamma, beta, yp, stats, part, batch, cut, dtype, eps, act, s);
}

template <typename T, int ACT, bool ONCE>
int cut_bwd(const T* dy, const T* x, const float* gamma, const float* beta, const double* stats, T* dx, float* dgamma,
            float* dbeta, float* part, long batch, const Cut& cut, int dtype, hipStream_t s) {
  float* sums = part + batch * cut.nchunk * cut.C * 2;
  float* coef = sums + batch * cut.C * 2;
  const dim3 grid((unsigned)(batch * cut.nchunk)), block(block_of(cut));
  const size_t lds = 2 * sizeof(float) * slots_of(cut, dtype);
  if (ONCE && cut.iters > GN_RUN) {
    if (int rc = allow_lds<gn_bwd_sums_kernel<T, ACT, true, true>>(lds)) return rc;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, ACT, true, true>), grid, block, lds, s, dy, x, gamma, beta, stats, cut, part);
  } else {
    if (int rc = allow_lds<gn_bwd_sums_kernel<T, ACT, ONCE, false>>(lds)) return rc;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, ACT, ONCE, false>), grid, block, lds, s, dy, x, gamma, beta, stats, cut, part);
  }
  const int span = cut.Cg > 64 ? 64 : 64 / cut.Cg * cut.Cg;
  hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)(batch * mmsa_cdiv(cut.C, span))),
                     dim3(cut.nchunk < 64 ? 256 : 1024), 0, s, part, cut, span, gamma, sums, coef);
  if (cut.Cg > 64 && dx)
    hipLaunchKernelGGL(gn_bwd_coef_kernel, dim3((unsigned)(batch * cut.G)), dim3(256), 0, s, sums, cut, gamma, coef);
  const int nparam = dgamma || dbeta ? mmsa_cdiv(cut.C, 64) : 0;
  const unsigned blocks = nparam + (dx ? grid.x : 0);
  if (blocks)
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, ACT, ONCE>), dim3(blocks), block, 0, s, dy, x, gamma, beta, stats, sums,
                       coef, dx, dgamma, dbeta, nparam, batch, cut);
  return mmsa_launch_status();
}

template <typename T, int ACT>
int gn_bwd(const void* dy, const void* x, const float* gamma, const float* beta, const double* stats, void* dx,
           float* dgamma, float* dbeta, void* scratch, long batch, const Cut& cut, int dtype, hipStream_t s) {
  float* part = static_cast<float*>(scratch);
  Slab q;
  if (make_slab(batch, cut.S / cut.C, cut.C, cut.G, dtype, BWD_REGS, true, &q)) {
    if (q.W == Io<T>::V)
      return slab_bwd_n<T, Io<T>::V, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, part, q, s);
    if constexpr (sizeof(T) == 2)
      if (q.W == 4) return slab_bwd_n<T, 4, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, part, q, s);
    if constexpr (sizeof(T) == 4)
      if (q.W == 2) return slab_bwd_n<T, 2, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, part, q, s);
    return slab_bwd_n<T, 1, ACT>(dy, x, gamma, beta, stats, dx, dgamma, dbeta, part, q, s);
  }
  const T* xp = static_cast<const T*>(x);
  const T* gp = static_cast<const T*>(dy);
  T* op = static_cast<T*>(dx);
  if (2 * batch * cut.S * (long)sizeof(T) > GN_CACHED || cut.iters > GN_RUN)
    return cut_bwd<T, ACT, true>(gp, xp, gamma, beta, stats, op, dgamma, dbeta, part, batch, cut, dtype, s);
  return cut_bwd<T, ACT, false>(gp, xp, gamma, beta, stats, op, dgamma, dbeta, part, batch, cut, dtype, s);
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
  // the joining kernels have a block of at most 256 threads per group, or per 64 channels (1024 only beside many chunks)
  const int most = groups > mmsa_cdiv(channels, 64) ? groups : mmsa_cdiv(channels, 64);
  if (batch > GN_MAX_BLOCKS / cut->nchunk || batch > 4 * GN_MAX_BLOCKS / most) return MMSA_ERR_LIMIT;
  return MMSA_OK;
}

}  // namespace

// Bytes of scratch the forward or the backward pass needs for these sizes (8-byte aligned; 0: none, it may be null).
MMSA_EXPORT long mmsa_group_norm_act_scratch_bytes(long batch, long positions, int channels, int groups, int dtype,
                                                   int backward) {
  Cut cut;
  Slab q;
  if (int rc = check_size(batch, positions, channels, groups, dtype, &cut)) return rc;
  if (make_slab(batch, positions, channels, groups, dtype, backward ? BWD_REGS : FWD_REGS, backward, &q))
    return backward ? batch * channels * 2 * 4 : 0;
  if (backward) return (batch * cut.nchunk * channels + batch * channels + batch * groups) * 2 * 4;
  return (batch * cut.nchunk * groups * 3 + batch * groups * 2) * 8;      // with a place for unwanted statistics
}

// y = act(group_norm(x) gamma + beta); stats [batch][groups][2] <- mean, 1 / sqrt(var + eps) in double, null: not wanted
MMSA_EXPORT int mmsa_group_norm_act_fwd(const void* x, const float* gamma, const float* beta, void* y, double* stats,
                                        void* scratch, long batch, long positions, int channels, int groups, float eps,
                                        int act, int dtype, void* stream) {
  MMSA_REQUIRE(x && y && act >= 0 && act <= 3 && eps >= 0.f);
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
