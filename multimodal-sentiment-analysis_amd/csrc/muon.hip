// Orthogonalised updates of weight matrices (Newton-Schulz products) and the Muon optimiser step built on them.
//
//   X_0 = u / max(||u||_F, eps)          (u^T where u has more rows than columns: X is [m][n] with m <= n)
//   X <- (a I + b S + c S S) X,  S = X X^T,   `steps` times, (a, b, c) = (3.4445, -4.775, 2.0315)
//     = B X,  B = (a - b^2 / 4c) I + c T T,  T = S + (b / 2c) I
// and for the optimiser   m <- m + (1 - mu)(g - m),  u = nesterov ? g + mu (m - g) : m,
//   p <- p (1 - lr wd) - lr max(1, rows / cols)^1/2 X_steps.
//
// Arithmetic.  x -> a x + b x^3 + c x^5 maps [0, 1.2025] into itself, so singular values, hence entries, of X never
// exceed 1.2025, those of T 1.18 and those of B 3.4445: every operand fits ONE fixed power-of-two
// scale of 2^14 in fp16, with no overflow for any input.  Each value is held as a pair hi = fp16(v), lo = fp16(v - hi),
// which is within 2^-23 of it (one unit of fp32 in a quarter of all values, exact in the others) or 2^-39 absolutely,
// and each product is three fp16 matrix products hi hi + hi lo + lo hi into fp32 accumulators.  lo lo is left out: at
// most 2^-22 of a product, of either sign, except on the diagonals of X X^T and T T, where it is a square and leaves
// them 2^-24.6 short in the mean.  Against 64 bits the result is off by 0.5 to 1.3 times what plain fp32 products leave
// (0.9 in the median of 151 matrices of 2 to 3000 rows; 1.4 with tiles of 256; for a handful of rows chance decides, up
// to 2.3), at a third of the fp16 matrix rate (about 2.5 PFLOP/s) instead of the fp32 matrix rate (157 TFLOP/s).
// A matrix whose norm is below eps enters with entries far below 1: its X is held at a larger scale 2^(14 + k), k from
// the norm (the polynomial grows it by at most a per step, so k shrinks from step to step by the same bound).
//
// The rule and the coefficients are published: K. Jordan and others, "Muon: an optimizer for hidden layers in neural
// networks" (2024).
//
// Layout.  A padded matrix [rows][K] of pairs is stored as [row][K / 16][hi 16 | lo 16] fp16: 16 values of a row, what
// one matrix instruction takes, are 64 bytes holding both halves.  All products are row times row
// (both operands K-contiguous): X X^T, T T (T is symmetric), and B X = B (X^T)^T, for which X^T is kept beside X.
// Padding rows and columns hold zeros and stay zero.
#include "mmsa_common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <string.h>

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float NS_A = 3.4445f, NS_C = 2.0315f;
// b S + c S S = c T T - b^2 / 4c with T = S + b / 2c: one matrix is stored instead of S, and B needs no second operand
constexpr float NS_SHIFT = (float)(-4.775 / (2.0 * 2.0315)), NS_REST = (float)(3.4445 - 4.775 * 4.775 / (4.0 * 2.0315));
constexpr int NS_SCALE = 14;           // log2 of the fixed-point scale
constexpr int MAX_STEPS = 16;
constexpr int GROUP = 24;              // matrices of one launch at most (their descriptors travel as kernel arguments)

enum { PH_SUMSQ = 0, PH_SPLIT = 1, PH_PRODUCT = 2 /* T, B, X */, PH_JOIN = 5 /* T, B */, PH_COUNT = 7 };

struct Mat {
  const void* g;        // gradient / input matrix, [rows][cols]
  void* out;            // orthogonalised matrix (same type as g) or the parameter (fp32), [rows][cols]
  float* mom;           // momentum buffer, or null
  char* ws;             // this matrix's part of the scratch
  long ws_off;
  int rows, cols;
  int m, n;             // the smaller and the larger of the two
  int mp, np;           // padded to the tile
  int part0, nparts;    // its partial sums of squares, `chunk` values each
  int chunk;
  int nsplit[2];        // blocks that share the K range of a tile of T / B
  float adjust;         // max(1, rows / cols)^1/2
};
// The descriptors of one set of launches: an argument of the first kernel, which leaves them at the start of the
// scratch for the others (an argument of this size costs the host a few microseconds per launch).
struct Group {
  Mat mat[GROUP];
  int first[PH_COUNT][GROUP];   // first block of every matrix in each kind of launch
  int count;
  int even[3];                  // all blocks of the T, B, X product have the same K
};
static_assert(sizeof(Group) < 4096 - 256, "kernel arguments are limited to 4 KiB");

// scratch of one matrix: X [mp][np], X^T [np][mp] twice (read and written in turn), T and B [mp][mp], k per step, the
// partial tiles of a split product
__host__ __device__ inline long row_bytes(long K) { return 4 * K; }
__host__ __device__ inline long xbytes(const Mat& q) { return q.mp * row_bytes(q.np); }
__host__ __device__ inline long tbytes(const Mat& q) { return q.np * row_bytes(q.mp); }
__host__ __device__ inline long sbytes(const Mat& q) { return q.mp * row_bytes(q.mp); }
__host__ __device__ inline long mat_bytes(const Mat& q) { return xbytes(q) + 2 * tbytes(q) + 2 * sbytes(q) + 128; }
__device__ __forceinline__ char* ws_x(const Mat& q) { return q.ws; }
__device__ __forceinline__ char* ws_xt(const Mat& q, int which) { return q.ws + xbytes(q) + which * tbytes(q); }
__device__ __forceinline__ char* ws_t(const Mat& q) { return q.ws + xbytes(q) + 2 * tbytes(q); }
__device__ __forceinline__ char* ws_b(const Mat& q) { return q.ws + xbytes(q) + 2 * tbytes(q) + sbytes(q); }
__device__ __forceinline__ int* ws_k(const Mat& q) { return reinterpret_cast<int*>(q.ws + mat_bytes(q) - 128); }
__device__ __forceinline__ float* ws_part(const Mat& q) { return reinterpret_cast<float*>(q.ws + mat_bytes(q)); }

// Which matrix a block works on: the last one whose first block is not behind it (all lanes of a wave call it).  `count`
// is a kernel argument, as is all that a block needs before it can ask for its descriptor: every load that waits for
// another one here is a microsecond of every launch.
__device__ __forceinline__ int find_mat(const int* first, int count, int block) {
  if (count == 1) return 0;
  const int lane = threadIdx.x & 63;
  const bool at_or_behind = first[lane < GROUP ? lane : 0] <= block && lane < count;
  // matrices without a block in this launch share their first block with the next one that has some
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(at_or_behind)) - 1);
}

// ---- element types
// four values at any alignment of one value (this target's global accesses allow it)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(2)));
template <typename T> struct El;
template <> struct El<float> {
  static __device__ __forceinline__ float get(const void* p, long i) { return static_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ f32x4 get4(const void* p, long i) {
    const f32x4u u = *reinterpret_cast<const f32x4u*>(static_cast<const float*>(p) + i);
    return f32x4{u[0], u[1], u[2], u[3]};
  }
  static __device__ __forceinline__ void put(void* p, long i, float v) { static_cast<float*>(p)[i] = v; }
  static __device__ __forceinline__ void put4(void* p, long i, f32x4 v) {
    f32x4u u = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4u*>(static_cast<float*>(p) + i) = u;
  }
};
template <> struct El<__hip_bfloat16> {
  static __device__ __forceinline__ float get(const void* p, long i) {
    return __uint_as_float((unsigned)static_cast<const unsigned short*>(p)[i] << 16);
  }
  static __device__ __forceinline__ f32x4 get4(const void* p, long i) {
    const u32x2u u = *reinterpret_cast<const u32x2u*>(static_cast<const unsigned short*>(p) + i);
    return f32x4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
                 __uint_as_float(u[1] & 0xffff0000u)};
  }
  static __device__ __forceinline__ void put(void* p, long i, float v) {
    static_cast<__hip_bfloat16*>(p)[i] = __float2bfloat16(v);
  }
  static __device__ __forceinline__ void put4(void* p, long i, f32x4 v) {
    __hip_bfloat16 h[4] = {__float2bfloat16(v[0]), __float2bfloat16(v[1]), __float2bfloat16(v[2]), __float2bfloat16(v[3])};
    u32x2u u;
    __builtin_memcpy(&u, h, 8);
    *reinterpret_cast<u32x2u*>(static_cast<__hip_bfloat16*>(p) + i) = u;
  }
};
template <> struct El<_Float16> {
  static __device__ __forceinline__ float get(const void* p, long i) {
    return (float)static_cast<const _Float16*>(p)[i];
  }
  static __device__ __forceinline__ f32x4 get4(const void* p, long i) {
    const u32x2u u = *reinterpret_cast<const u32x2u*>(static_cast<const _Float16*>(p) + i);
    _Float16 h[4];
    __builtin_memcpy(h, &u, 8);
    return f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
  }
  static __device__ __forceinline__ void put(void* p, long i, float v) { static_cast<_Float16*>(p)[i] = (_Float16)v; }
  static __device__ __forceinline__ void put4(void* p, long i, f32x4 v) {
    _Float16 h[4] = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    u32x2u u;
    __builtin_memcpy(&u, h, 8);
    *reinterpret_cast<u32x2u*>(static_cast<_Float16*>(p) + i) = u;
  }
};

__device__ __forceinline__ float direction(float g, float mom, float mu, int nesterov) {
  return nesterov ? fmaf(mu, mom - g, g) : mom;
}

// Momentum update (MOM) and the sum of squares of u in 64 bits, one block per chunk; bound by memory: 33.6 M values in
// five matrices 72 us, 402 MB at 5.6 TB/s.
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void momentum_sumsq_kernel(const Group gr, float mu, float one_minus_mu, int nesterov,
                                                             double* __restrict__ parts, Group* __restrict__ dev) {
  __shared__ double red[16];
  if (blockIdx.x == 0) {
    const int* from = reinterpret_cast<const int*>(&gr);
    for (int j = threadIdx.x; j < (int)(sizeof(Group) / 4); j += 256) reinterpret_cast<int*>(dev)[j] = from[j];
  }
  const int i = find_mat(gr.first[PH_SUMSQ], gr.count, blockIdx.x);
  const Mat& q = gr.mat[i];
  const int c = blockIdx.x - gr.first[PH_SUMSQ][i];
  const long lo = (long)c * q.chunk, total = (long)q.rows * q.cols;
  const int n = (int)(total - lo < q.chunk ? total - lo : q.chunk), n4 = n & ~3;
  const T* g = static_cast<const T*>(q.g) + lo;
  float* mom = MOM ? q.mom + lo : nullptr;
  double ss = 0.0;
#pragma unroll 4
  for (int j = 4 * threadIdx.x; j < n4; j += 1024) {
    f32x4 u = El<T>::get4(g, j);
    if (MOM) {
      f32x4u m = *reinterpret_cast<const f32x4u*>(mom + j);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[k] = fmaf(one_minus_mu, u[k] - m[k], m[k]);
        u[k] = direction(u[k], m[k], mu, nesterov);
      }
      *reinterpret_cast<f32x4u*>(mom + j) = m;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) ss += (double)u[k] * (double)u[k];
  }
  if ((int)threadIdx.x < n - n4) {
    const int j = n4 + threadIdx.x;
    float u = El<T>::get(g, j);
    if (MOM) {
      const float m = fmaf(one_minus_mu, u - mom[j], mom[j]);
      mom[j] = m;
      u = direction(u, m, mu, nesterov);
    }
    ss += (double)u * (double)u;
  }
  ss = block_sum_d(ss, red);
  if (threadIdx.x == 0) parts[q.part0 + c] = ss;
}

__device__ __forceinline__ void put_pair(char* base, long row, long col, long K, float v) {
  const _Float16 hi = (_Float16)v;
  _Float16* p = reinterpret_cast<_Float16*>(base + row * row_bytes(K)) + (col >> 4) * 32 + (col & 15);
  p[0] = hi;
  p[16] = (_Float16)(v - (float)hi);
}

// how far X's scale exceeds 2^NS_SCALE for a bound r on its norm
__device__ __forceinline__ int extra_scale(double r) {
  if (!(r > 0.0) || r >= 1.0) return 0;
  return min(400, max(0, (int)floor(-log2(r))));
}

// normalises u and writes X and X^T as pairs, 64 x 64 values of u's padded extent per block, 16 bytes a lane: sixteen
// lanes write 256 consecutive bytes of a row.  Bound by memory: 33.6 M values with momentum 101 us, 537 MB at 5.3 TB/s.
// Every block adds up the (at most 512) partial sums of its matrix itself, which spares a launch.
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void split_kernel(const Group* __restrict__ grp, int count, float mu, int nesterov, float eps,
                                                    int steps, const double* __restrict__ parts) {
  __shared__ double red[16];
  __shared__ float tile[64][65];
  const Group& gr = *grp;
  const int i = find_mat(gr.first[PH_SPLIT], count, blockIdx.x);
  const Mat& q = gr.mat[i];
  const int b = blockIdx.x - gr.first[PH_SPLIT][i];
  const bool tall = q.rows > q.cols;
  const int pr = tall ? q.np : q.mp, pc = tall ? q.mp : q.np;      // padded extent in u's own orientation
  const int nct = pc / 64;
  const long r0 = (long)(b / nct) * 64, c0 = (long)(b % nct) * 64;
  // the values first, so that they arrive while the norm is added up
  float u[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const long row = r0 + (threadIdx.x >> 4) + 16 * k, col = c0 + (threadIdx.x & 15) * 4;
    const long at = row * q.cols + col;
    const int n = row >= q.rows || col >= q.cols ? 0 : q.cols - col < 4 ? (int)(q.cols - col) : 4;
    if (n == 4) {
      const f32x4 v = El<T>::get4(q.g, at);
      f32x4u m{};
      if (MOM) m = *reinterpret_cast<const f32x4u*>(q.mom + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[k][e] = MOM ? direction(v[e], m[e], mu, nesterov) : v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[k][e] = 0.f;
        if (e < n) {
          u[k][e] = El<T>::get(q.g, at + e);
          if (MOM) u[k][e] = direction(u[k][e], q.mom[at + e], mu, nesterov);
        }
      }
    }
  }
  double ss = 0.0;
  for (int j = threadIdx.x; j < q.nparts; j += 256) ss += parts[q.part0 + j];
  ss = block_sum_d(ss, red);
  const double norm = sqrt(ss);
  const double size = norm > (double)eps ? norm : (norm != norm ? norm : (double)eps);
  double r = norm / size;
  const int k0 = extra_scale(r);
  if (b == 0 && threadIdx.x == 0) {
    int* k = ws_k(q);
    for (int t = 0; t <= steps; ++t) {
      k[t] = extra_scale(r);
      r = fmin((double)NS_A * r, 1.2025);
    }
  }
  const double mul = ldexp(1.0 / size, NS_SCALE + k0);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      tile[(threadIdx.x >> 4) + 16 * k][(threadIdx.x & 15) * 4 + e] = (float)((double)u[k][e] * mul);
  __syncthreads();
  char* rowm = tall ? ws_xt(q, 0) : ws_x(q);                       // [pr][pc]
  char* colm = tall ? ws_x(q) : ws_xt(q, 0);                       // [pc][pr]
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int line = (threadIdx.x >> 4) + 16 * k, unit = threadIdx.x & 15;
    const int at = (unit >> 2) * 16 + (unit & 1) * 8;              // units of a run: hi, hi, lo, lo
    f16x8 o, t;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = tile[line][at + e], c = tile[at + e][line];
      const _Float16 hv = (_Float16)v, hc = (_Float16)c;
      o[e] = unit & 2 ? (_Float16)(v - (float)hv) : hv;
      t[e] = unit & 2 ? (_Float16)(c - (float)hc) : hc;
    }
    *reinterpret_cast<f16x8*>(rowm + (r0 + line) * row_bytes(pc) + c0 * 4 + unit * 16) = o;
    *reinterpret_cast<f16x8*>(colm + (c0 + line) * row_bytes(pr) + r0 * 4 + unit * 16) = t;
  }
}

// ---- products
enum { TO_T = 0, TO_B = 1, TO_X = 2, TO_OUT = 3, TO_PARAM = 4 };

// 16 bytes per lane straight into LDS: lane l of the wave lands at lds + 16 l
__device__ __forceinline__ void load_lds16(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

__device__ __forceinline__ void lower_tile(int b, int& ti, int& tj) {
  ti = (int)((sqrtf(8.f * (float)b + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
  while (ti * (ti + 1) / 2 > b) --ti;
  tj = b - ti * (ti + 1) / 2;
}

// factor of the accumulator in the stored result, and what is added to the diagonal
template <int MODE>
__device__ __forceinline__ float result_scale(const Mat& q, int step) {
  const int k0 = ws_k(q)[step], k1 = ws_k(q)[step + 1];
  return MODE == TO_T   ? ldexpf(1.f, -NS_SCALE - 2 * k0)
         : MODE == TO_B ? ldexpf(NS_C, -NS_SCALE)
         : MODE == TO_X ? ldexpf(1.f, k1 - k0 - NS_SCALE)
                        : ldexpf(1.f, -2 * NS_SCALE - k0);
}
template <int MODE>
__device__ __forceinline__ float diagonal() {
  return ldexpf(MODE == TO_T ? NS_SHIFT : NS_REST, NS_SCALE);
}

// The order in which tiles are given to blocks: consecutive blocks go to the eight XCDs in turn, each with an L2 of its
// own, so every XCD gets one consecutive run of tiles (whose operand rows it shares) -- of all the launch's tiles where
// they take equally long, else of every matrix's, so that no XCD gets the long ones.
__device__ __forceinline__ int xcd_order(int l, int n) {
  const int per = n >> 3;
  return l < per << 3 ? (l & 7) * per + (l >> 3) : l;
}

// Shape of a product block: BT x BT outputs, four waves as 2 x 2, each with W x W tiles of 32 x 32.
template <int BT>
struct Tile {
  static constexpr int W = BT / 64;
  static constexpr int G = BT == 256 ? 1 : 2;         // groups of 16 values of K in a step
  static constexpr int ROW = 64 * G;                    // bytes of an operand row in one LDS buffer
  static constexpr int OPER = BT * ROW;
  static constexpr int RING = 4;                        // LDS buffers
  static constexpr int LOADS = BT * G / 32;             // a thread's loads per step
  static constexpr int SUMS = BT == 256 ? 1 : 2;        // accumulators per value
  static constexpr int PASSES = BT == 256 ? 2 : 1;      // rounds in which the results leave through LDS
  static constexpr int OUTROW = BT * 4 + 16;            // an output row of pairs in LDS, padded against bank conflicts
  static constexpr int LDS = RING * 2 * OPER > BT / PASSES * OUTROW ? RING * 2 * OPER : BT / PASSES * OUTROW;
};

// waits until at most N of this wave's global loads are on their way (they return in order) and its LDS reads are done,
// then for the other waves
template <int N>
__device__ __forceinline__ void wait_loads_and_meet() {
  static_assert(N >= 0 && N < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// acc += P Q^T over nk32 * 32 values.  Each wave runs ahead of itself: a ring of four LDS buffers, loads straight into LDS
// issued three steps ahead and waited for by count, and the fragments of the next step read while the matrix
// instructions of this one run, one load or read between two of them.  The 16-byte units of a row are XORed with bits of
// the row, which makes the fragment reads free of bank conflicts: 16 lanes of one read cover the 16 units of 256 bytes.
template <int BT>
struct Fragments {
  f16x8 ph[Tile<BT>::G][Tile<BT>::W], pl[Tile<BT>::G][Tile<BT>::W];
  f16x8 qh[Tile<BT>::G][Tile<BT>::W], ql[Tile<BT>::G][Tile<BT>::W];
};

//
// A matrix instruction rounds twice into its fp32 accumulator.  The products hi lo + lo hi are 2^-11 of hi hi: in an
// accumulator of their own they round at that scale, and the main one is rounded a third as often (0.6 of the error at
// K = 2048).  The 256 x 256 tile has no registers left for that: four 2048 x 2048 and a 2048 x 8192 end 1.2 to 1.4 times as
// far from the exact result as plain fp32 products do.
template <int BT>
__device__ __forceinline__ void multiply(f32x16 (&acc)[Tile<BT>::W][Tile<BT>::W], char* lds, const char* P,
                                         const char* Q, long pitch, int nk32) {
  typedef Tile<BT> S;
  f32x16 low[S::SUMS == 2 ? S::W : 1][S::SUMS == 2 ? S::W : 1];
  if (S::SUMS == 2) {
#pragma unroll
    for (int x = 0; x < (S::SUMS == 2 ? S::W : 1); ++x)
#pragma unroll
      for (int y = 0; y < (S::SUMS == 2 ? S::W : 1); ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) low[x][y][e] = 0.f;
  }
  constexpr int W = S::W, G = S::G, ROW = S::ROW, OPER = S::OPER, LOADS = S::LOADS;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);     // LDS places in scalars
  const int nk = nk32 * 2 / G;
  // a wave's load fills 16 / G rows
  const int lrow = lane / (4 * G), lu = lane % (4 * G);
  const int lunit = lu ^ (G == 1 ? (lrow >> 2) & 3 : ((w & 1) * 4 + (lrow >> 1)) & 7);
  const char* ps = P + (w * (16 / G) + lrow) * pitch + lunit * 16;
  const char* qs = Q + (w * (16 / G) + lrow) * pitch + lunit * 16;
  auto stage = [&](int k) {
    char* to = lds + (k & 3) * 2 * OPER + w * 1024;
#pragma unroll
    for (int j = 0; j < LOADS / 2; ++j) {
      load_lds16(ps + j * (64 / G) * pitch + (long)k * ROW, to + j * 4096);
      load_lds16(qs + j * (64 / G) * pitch + (long)k * ROW, to + OPER + j * 4096);
    }
  };
  const int fr = lane & 31, half = lane >> 5, swz = G == 1 ? (fr >> 2) & 3 : (fr >> 1) & 7;
  const int prow = ((w >> 1) * W * 32 + fr) * ROW, qrow = OPER + ((w & 1) * W * 32 + fr) * ROW;
  auto fetch = [&](Fragments<BT>& f, int k) {
    const char* l0 = lds + (k & 3) * 2 * OPER;
#pragma unroll
    for (int s = 0; s < G; ++s) {
      const int uh = ((s * 4 + half) ^ swz) * 16, ul = ((s * 4 + 2 + half) ^ swz) * 16;
#pragma unroll
      for (int x = 0; x < W; ++x) {
        f.qh[s][x] = *reinterpret_cast<const f16x8*>(l0 + qrow + x * 32 * ROW + uh);
        f.ql[s][x] = *reinterpret_cast<const f16x8*>(l0 + qrow + x * 32 * ROW + ul);
        f.ph[s][x] = *reinterpret_cast<const f16x8*>(l0 + prow + x * 32 * ROW + uh);
        f.pl[s][x] = *reinterpret_cast<const f16x8*>(l0 + prow + x * 32 * ROW + ul);
      }
    }
  };
  auto compute = [&](const Fragments<BT>& f) {
#pragma unroll
    for (int s = 0; s < G; ++s)
#pragma unroll
      for (int x = 0; x < W; ++x) {
#pragma unroll
        for (int y = 0; y < W; ++y) {
          f32x16& to = S::SUMS == 2 ? low[S::SUMS == 2 ? x : 0][S::SUMS == 2 ? y : 0] : acc[x][y];
          to = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.pl[s][x], f.qh[s][y], to, 0, 0, 0);
        }
#pragma unroll
        for (int y = 0; y < W; ++y) {
          f32x16& to = S::SUMS == 2 ? low[S::SUMS == 2 ? x : 0][S::SUMS == 2 ? y : 0] : acc[x][y];
          to = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[s][x], f.ql[s][y], to, 0, 0, 0);
        }
#pragma unroll
        for (int y = 0; y < W; ++y)
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[s][x], f.qh[s][y], acc[x][y], 0, 0, 0);
      }
  };
  auto join = [&]() {
    if (S::SUMS == 1) return;
#pragma unroll
    for (int x = 0; x < (S::SUMS == 2 ? W : 0); ++x)
#pragma unroll
      for (int y = 0; y < (S::SUMS == 2 ? W : 0); ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[x][y][e] += low[x][y][e];
  };
  // Step k: step k + 1 has arrived for all waves, so its fragments can be read; the buffer of step k + 3 held step
  // k - 1, whose fragments every wave had before it came here.  The reads and loads are spread over the matrix
  // instructions, none of which depends on them.
  auto step = [&](const Fragments<BT>& now, Fragments<BT>& next, int k) {
    wait_loads_and_meet<LOADS>();
    stage(k + 3);
    fetch(next, k + 1);
    compute(now);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);            // matrix
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);            // global load
    }
#pragma unroll
    for (int i = 0; i < 4 * W * G; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);            // matrix
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);            // LDS read
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // nk is even
  Fragments<BT> a, b;
  stage(0);
  stage(1);
  if (nk == 2) {
    wait_loads_and_meet<0>();
    fetch(a, 0);
    fetch(b, 1);
    compute(a);
    compute(b);
    join();
    return;
  }
  stage(2);
  wait_loads_and_meet<2 * LOADS>();
  fetch(a, 0);
  int k = 0;
  for (; k + 4 < nk; k += 2) {
    step(a, b, k);
    step(b, a, k + 1);
  }
  step(a, b, k);
  wait_loads_and_meet<0>();
  fetch(a, k + 2);
  compute(b);
  __builtin_amdgcn_sched_barrier(0);
  fetch(b, k + 3);
  compute(a);
  __builtin_amdgcn_sched_barrier(0);
  compute(b);
  join();
}

// D = P Q^T for one BT x BT tile of one matrix.  Measured (three fp16 products each):
//   256 tile, X of four 2048 x 2048 and one 2048 x 8192: 404 us, 1.02 PFLOP/s (a library fp16 product of 8192^3: 1.23)
//   128 tile, X of 1024 x 4096: 32 us, 0.8 PFLOP/s; T of the five above: 229 us, 0.96
//   64 tile, X of 1023 x 1537: 19 us; T: 16.5 us, of which 4 are the start and the end of a block
// The loads bound the two smaller tiles: T of the five takes 143 us without them, 196 without matrix instructions.  A
// compute unit keeps about 75 lines of 128 bytes on their way, at 400 clocks each (a third of them lie behind another
// XCD's L2, whose blocks wrote them in the launch before), which is 60 GB/s; a deeper ring does not change that.
// T and B are symmetric: only tiles on and below the diagonal are computed, the others are written as their mirror
// image.  Where a phase has few tiles and a long K, a share of the K steps goes to one block each and the partial
// results meet in join_kernel.
template <typename T, int BT, int MODE>
__global__ __launch_bounds__(256, BT == 256 || Tile<BT>::LDS > 81920 ? 1 : 2) void product_kernel(
    const Group* __restrict__ grp, int count, int even, int step, int which, float decay, float rate) {
  typedef Tile<BT> S;
  constexpr int W = S::W;
  __shared__ __attribute__((aligned(128))) char lds[S::LDS];
  const Group& gr = *grp;
  constexpr int PHASE = MODE < TO_X ? MODE : TO_X;
  const int block = even ? xcd_order(blockIdx.x, gridDim.x) : blockIdx.x;
  const int mi = find_mat(gr.first[PH_PRODUCT + PHASE], count, block);
  const Mat& q = gr.mat[mi];
  const int b = block - gr.first[PH_PRODUCT + PHASE][mi];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int K = MODE == TO_T ? q.np : q.mp;
  int ti, tj, k_lo = 0, nk = K / 32, part = 0, nsplit = 1, tile = 0;
  if (MODE <= TO_B) {
    const int nt = q.mp / BT;
    nsplit = q.nsplit[PHASE];
    const int l = even ? b : xcd_order(b, nt * (nt + 1) / 2 * nsplit);
    tile = l / nsplit;
    part = l % nsplit;
    lower_tile(tile, ti, tj);
    const int kper = ((nk >> 1) + nsplit - 1) / nsplit * 2;      // an even number of steps
    k_lo = part * kper;
    nk = nk - k_lo < kper ? nk - k_lo : kper;
  } else {
    // bands of eight tile rows, column by column
    const int mt = q.mp / BT, nt = q.np / BT;
    const int l = even ? b : xcd_order(b, mt * nt);
    const int band = l / (8 * nt), rows = mt - band * 8 < 8 ? mt - band * 8 : 8, r = l - band * 8 * nt;
    ti = band * 8 + r % rows;
    tj = r / rows;
  }
  const char* P = MODE == TO_T ? ws_x(q) : MODE == TO_B ? ws_t(q) : ws_b(q);
  const char* Q = MODE == TO_T ? ws_x(q) : MODE == TO_B ? ws_t(q) : ws_xt(q, which);
  const long pitch = row_bytes(K);
  f32x16 acc[W][W];
#pragma unroll
  for (int x = 0; x < W; ++x)
#pragma unroll
    for (int y = 0; y < W; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  multiply<BT>(acc, lds, P + (long)ti * BT * pitch + k_lo * 128l, Q + (long)tj * BT * pitch + k_lo * 128l, pitch, nk);
  const int wi = w >> 1, wj = w & 1, fr = lane & 31, half = lane >> 5;
  // register e of a wave's tile (x, y): row (e & 3) + 8 (e >> 2) + 4 half, column fr
  if (MODE <= TO_B && nsplit > 1) {
    float* o = ws_part(q) + ((long)tile * nsplit + part) * (BT * BT) + tid;
#pragma unroll
    for (int x = 0; x < W; ++x)
#pragma unroll
      for (int y = 0; y < W; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[((x * W + y) * 16 + e) * 256] = acc[x][y][e];
    return;
  }
  const float mul = result_scale<MODE>(q, step);
  const int i0 = wi * W * 32 + 4 * half, j0 = wj * W * 32 + fr;
  // the tile and its transpose leave through LDS as rows of pairs, 16 bytes a lane
  const bool diag = MODE <= TO_B && ti == tj;
#pragma unroll
  for (int x = 0; x < W; ++x)
#pragma unroll
    for (int y = 0; y < W; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] *= mul;
  constexpr int ROWS = BT / S::PASSES;
  if (MODE >= TO_OUT) {
    // results in the orientation of the caller's matrix, as rows of floats through LDS
    const bool tall = q.rows > q.cols;
    const long row0 = (long)(tall ? tj : ti) * BT, col0 = (long)(tall ? ti : tj) * BT;
#pragma unroll
    for (int p = 0; p < S::PASSES; ++p) {
      __syncthreads();
      if (S::PASSES == 1 || (tall ? j0 : i0) / ROWS == p) {
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
          for (int y = 0; y < W; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int i = i0 + x * 32 + 8 * g, j = j0 + y * 32;
              if (tall) {
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[x][y][g * 4 + r];
                *reinterpret_cast<f32x4*>(lds + (j - p * ROWS) * S::OUTROW + i * 4) = v;
              } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  *reinterpret_cast<float*>(lds + (i + r - p * ROWS) * S::OUTROW + j * 4) = acc[x][y][g * 4 + r];
              }
            }
      }
      __syncthreads();
      for (int u = tid; u < ROWS * BT / 4; u += 256) {
        const int r = u / (BT / 4), c = u % (BT / 4) * 4;
        const long row = row0 + p * ROWS + r, col = col0 + c;
        if (row >= q.rows || col >= q.cols) continue;
        const f32x4 v = *reinterpret_cast<const f32x4*>(lds + r * S::OUTROW + c * 4);
        const long at = row * q.cols + col;
        const int n = q.cols - col < 4 ? (int)(q.cols - col) : 4;
        if (MODE == TO_OUT) {
          if (n == 4)
            El<T>::put4(q.out, at, v);
          else
            for (int k = 0; k < n; ++k) El<T>::put(q.out, at + k, v[k]);
        } else {
          float* o = static_cast<float*>(q.out) + at;
          const float f = -rate * q.adjust;
          if (n == 4) {
            f32x4u old = *reinterpret_cast<const f32x4u*>(o);
#pragma unroll
            for (int k = 0; k < 4; ++k) old[k] = fmaf(old[k], decay, f * v[k]);
            *reinterpret_cast<f32x4u*>(o) = old;
          } else {
            for (int k = 0; k < n; ++k) o[k] = fmaf(o[k], decay, f * v[k]);
          }
        }
      }
    }
    return;
  }
  char* direct = MODE == TO_T ? ws_t(q) : MODE == TO_B ? ws_b(q) : ws_x(q);
  char* mirror = MODE == TO_X ? ws_xt(q, which ^ 1) : direct;
  const long dpitch = row_bytes(MODE == TO_X ? q.np : q.mp), mpitch = row_bytes(q.mp);
  auto copy_out = [&](char* dst, long dst_pitch) {
    for (int u = tid; u < ROWS * BT / 4; u += 256) {
      const int row = u / (BT / 4), unit = u % (BT / 4);
      *reinterpret_cast<uint4*>(dst + row * dst_pitch + unit * 16) =
          *reinterpret_cast<const uint4*>(lds + row * S::OUTROW + unit * 16);
    }
  };
#pragma unroll
  for (int p = 0; p < S::PASSES; ++p) {
    __syncthreads();
    if (S::PASSES == 1 || i0 / ROWS == p) {
#pragma unroll
      for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int i = i0 - p * ROWS + x * 32 + (e & 3) + 8 * (e >> 2), j = j0 + y * 32;
            const float v = acc[x][y][e];
            const _Float16 hi = (_Float16)v;
            _Float16* o = reinterpret_cast<_Float16*>(lds + i * S::OUTROW + (j >> 4) * 64) + (j & 15);
            o[0] = hi;
            o[16] = (_Float16)(v - (float)hi);
          }
    }
    __syncthreads();
    if (diag) {
      if (tid < ROWS) {
        const int j = p * ROWS + tid;
        _Float16* o = reinterpret_cast<_Float16*>(lds + tid * S::OUTROW + (j >> 4) * 64) + (j & 15);
        const float v = ((float)o[0] + (float)o[16]) + diagonal<MODE>();
        const _Float16 hi = (_Float16)v;
        o[0] = hi;
        o[16] = (_Float16)(v - (float)hi);
      }
      __syncthreads();
    }
    copy_out(direct + ((long)ti * BT + p * ROWS) * dpitch + tj * (BT * 4l), dpitch);
  }
  if (diag) return;
#pragma unroll
  for (int p = 0; p < S::PASSES; ++p) {
    __syncthreads();
    if (S::PASSES == 1 || j0 / ROWS == p) {
#pragma unroll
      for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int i = i0 + x * 32 + 8 * g, j = j0 - p * ROWS + y * 32;
            f16x4 hi, lo;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float v = acc[x][y][g * 4 + r];
              hi[r] = (_Float16)v;
              lo[r] = (_Float16)(v - (float)hi[r]);
            }
            char* o = lds + j * S::OUTROW + (i >> 4) * 64 + (i & 15) * 2;
            *reinterpret_cast<f16x4*>(o) = hi;
            *reinterpret_cast<f16x4*>(o + 32) = lo;
          }
    }
    __syncthreads();
    copy_out(mirror + ((long)tj * BT + p * ROWS) * mpitch + ti * (BT * 4l), mpitch);
  }
}

// Four values of T or B, rows i .. i + 3 of column j: scaled, as pairs, in their place and (outside the tiles of the
// diagonal) its mirror image.
template <int MODE>
__device__ __forceinline__ void store_four(const Mat& q, int step, const f32x4& v, long i, long j, bool mirrored) {
  const float mul = result_scale<MODE>(q, step);
  char* dst = MODE == TO_T ? ws_t(q) : ws_b(q);
  f16x4 hi, lo;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float o = v[k] * mul;
    if (i + k == j) o += diagonal<MODE>();
    hi[k] = (_Float16)o;
    lo[k] = (_Float16)(o - (float)hi[k]);
    put_pair(dst, i + k, j, q.mp, o);
  }
  if (!mirrored) return;
  char* o = dst + j * row_bytes(q.mp) + (i >> 4) * 64 + (i & 15) * 2;
  *reinterpret_cast<f16x4*>(o) = hi;
  *reinterpret_cast<f16x4*>(o + 32) = lo;
}

// T or B in tiles of 32 x 32, for matrices whose larger tiles would leave most compute units without one: a step is 64
// values of K, a quarter of it for each of the four waves, whose sums meet in LDS at the end.
// 700 x 700, 253 tiles instead of 66: 135 us for the five steps instead of 163; the model's twelve convolutions need no
// split of K for it, 140 us instead of 150.  Twice the bytes of a 64 tile per product: beyond a
// block per compute unit it loses (1024 x 1024: 528 blocks).
template <int MODE>
__global__ __launch_bounds__(256, 2) void narrow_kernel(const Group* __restrict__ grp, int count, int even,
                                                            int step) {
  constexpr int RING = 4, ROW = 256, OPER = 32 * ROW, BUF = 2 * OPER, LOADS = 4;
  __shared__ __attribute__((aligned(128))) char lds[RING * BUF];
  const Group& gr = *grp;
  const int block = even ? xcd_order(blockIdx.x, gridDim.x) : blockIdx.x;
  const int mi = find_mat(gr.first[PH_PRODUCT + MODE], count, block);
  const Mat& q = gr.mat[mi];
  const int b = block - gr.first[PH_PRODUCT + MODE][mi];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nt = q.mp / 32, nsplit = q.nsplit[MODE];
  const int l = even ? b : xcd_order(b, nt * (nt + 1) / 2 * nsplit), tile = l / nsplit, part = l % nsplit;
  int ti, tj;
  lower_tile(tile, ti, tj);
  const int K = MODE == TO_T ? q.np : q.mp, all = K / 64;
  const int kper = (all + nsplit - 1) / nsplit, k_lo = part * kper, nk = all - k_lo < kper ? all - k_lo : kper;
  const long pitch = row_bytes(K);
  const char* X = (MODE == TO_T ? ws_x(q) : ws_t(q)) + (long)k_lo * ROW;
  // a wave's load fills four rows; unit u of row r lies at u ^ (r & 15), so that 16 lanes of a fragment read cover all banks
  const int row = 4 * w + (lane >> 4);
  const char* ps = X + (ti * 32l + row) * pitch + ((lane & 15) ^ row) * 16;
  const char* qs = X + (tj * 32l + row) * pitch + ((lane & 15) ^ row) * 16;
  auto stage = [&](int k) {
    char* to = lds + (k & (RING - 1)) * BUF + w * 1024;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      load_lds16(ps + j * 16 * pitch + (long)k * ROW, to + j * 4096);
      load_lds16(qs + j * 16 * pitch + (long)k * ROW, to + OPER + j * 4096);
    }
  };
  const int fr = lane & 31, half = lane >> 5;
  const int uh = fr * ROW + ((4 * w + half) ^ (fr & 15)) * 16, ul = fr * ROW + ((4 * w + 2 + half) ^ (fr & 15)) * 16;
  f32x16 acc, low;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = low[e] = 0.f;
  for (int k = 0; k < RING - 1 && k < nk; ++k) stage(k);
  for (int k = 0; k < nk; ++k) {
    // the steps behind this one may still be on their way
    if (k + 2 < nk)
      wait_loads_and_meet<2 * LOADS>();
    else if (k + 1 < nk)
      wait_loads_and_meet<LOADS>();
    else
      wait_loads_and_meet<0>();
    if (k + RING - 1 < nk) stage(k + RING - 1);       // into the buffer of step k - 1, which all waves have read
    const char* l0 = lds + (k & (RING - 1)) * BUF;
    const f16x8 ph = *reinterpret_cast<const f16x8*>(l0 + uh), pl = *reinterpret_cast<const f16x8*>(l0 + ul);
    const f16x8 qh = *reinterpret_cast<const f16x8*>(l0 + OPER + uh), ql = *reinterpret_cast<const f16x8*>(l0 + OPER + ul);
    low = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, low, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, low, 0, 0, 0);
  }
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);          // [wave][register][lane]
#pragma unroll
  for (int e = 0; e < 16; ++e) sums[(w * 16 + e) * 64 + lane] = acc[e] + low[e];
  __syncthreads();
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float* p = sums + (4 * w + r) * 64 + lane;
    v[r] = (p[0] + p[1024]) + (p[2048] + p[3 * 1024]);
  }
  if (nsplit > 1) {
    float* o = ws_part(q) + ((long)tile * nsplit + part) * 1024 + 4 * w * 64 + lane;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r * 64] = v[r];
    return;
  }
  // register e of a lane: row (e & 3) + 8 (e >> 2) + 4 half, column fr
  store_four<MODE>(q, step, v, ti * 32l + 8 * w + 4 * half, tj * 32l + fr, ti != tj);
}

// Sums the partial tiles of the matrices whose K was split, four values (of one column) per lane: 4 to 8 us, nearly all of
// it the launch and a chain of three dependent loads; 15 us for the 2048 x 8192 one.  Many parts are shared
// out among a block's four waves; of few parts every wave adds up its own values.
__host__ __device__ inline bool many_parts(int nsplit) { return nsplit >= 8; }

template <int BT, int MODE>
__global__ __launch_bounds__(256) void join_kernel(const Group* __restrict__ grp, int count, int step) {
  constexpr int W = BT == 32 ? 1 : Tile<BT == 32 ? 64 : BT>::W, PER = BT * BT / 256;          // groups of 64 x 4 values in a tile
  constexpr int WAVES = BT == 32 ? 1 : 4, REG = 64 * WAVES;    // waves that hold a tile, values of one register of them
  __shared__ f32x4 sums[4][64];
  const Group& gr = *grp;
  const int mi = find_mat(gr.first[PH_JOIN + MODE], count, blockIdx.x);
  const Mat& q = gr.mat[mi];
  const int b = blockIdx.x - gr.first[PH_JOIN + MODE][mi], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nsplit = q.nsplit[MODE];
  const bool many = many_parts(nsplit);
  const int unit = many ? b : b * 4 + wave, tile = unit / PER, r = unit % PER;
  const int w = r % WAVES, g = r / WAVES & 3, x = r / (4 * WAVES) / W, y = r / (4 * WAVES) % W;
  const float* p = ws_part(q) + (long)tile * nsplit * (BT * BT) + ((x * W + y) * 16 + 4 * g) * REG + w * 64 + lane;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = many ? wave : 0; s < nsplit; s += many ? 4 : 1)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += p[(long)s * (BT * BT) + k * REG];
  if (many) {
    sums[wave][lane] = v;
    __syncthreads();
    if (wave) return;
    v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  }
  int ti, tj;
  lower_tile(tile, ti, tj);
  const long i = (long)ti * BT + (w >> 1) * W * 32 + x * 32 + 8 * g + 4 * (lane >> 5);
  const long j = (long)tj * BT + (w & 1) * W * 32 + y * 32 + (lane & 31);
  store_four<MODE>(q, step, v, i, j, ti != tj);
}

// ---- matrices that fit one block
// m <= 64 and n <= 32 * 8 * NT: the whole iteration in one launch, a block of eight waves per matrix.  At these sizes the
// seventeen dependent launches of the general path are all there is to its time (64 x 288, one matrix: 72 us, here 35).
// X lives in registers: wave w holds the column tiles w, w + 8, ... of 32 columns as the pairs that the product B X
// takes and gives back -- the accumulator of a product (lane: column; registers: rows 4 h + (e & 3) + 8 (e >> 2) of
// each 32) is the right operand of the next one with its K index in that order, and the left operand, B, is read from
// LDS in the same order.  X X^T needs X by rows: a wave turns its tiles over in LDS, and the waves' parts are added up
// there.  In LDS a pair is one 32-bit word, lo << 16 | hi.
constexpr int SMALL_M = 64;
constexpr int TURN_ROW = 36, SQUARE_ROW = 68;          // words of a row, padded against bank conflicts
constexpr int WAVE_WORDS = 3 * 16 * 64;                // a wave's part of X X^T: three of the four 32 x 32 tiles
static_assert(64 * TURN_ROW <= WAVE_WORDS, "a wave's turning buffer and its part of the sum share their place");

__device__ __forceinline__ unsigned to_pair(float v) {
  const _Float16 p[2] = {(_Float16)v, (_Float16)(v - (float)(_Float16)v)};
  unsigned u;
  __builtin_memcpy(&u, p, 4);
  return u;
}
// eight pairs -> the two fragments
__device__ __forceinline__ void from_pairs(const uint4& a, const uint4& b, f16x8& hi, f16x8& lo) {
  const unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  unsigned h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[k] = __builtin_amdgcn_perm(w[2 * k + 1], w[2 * k], 0x05040100);
    l[k] = __builtin_amdgcn_perm(w[2 * k + 1], w[2 * k], 0x07060302);
  }
  __builtin_memcpy(&hi, h, 16);
  __builtin_memcpy(&lo, l, 16);
}
// one product of pairs, the low ones in an accumulator of their own
__device__ __forceinline__ void pair_product(const f16x8& ph, const f16x8& pl, const f16x8& qh, const f16x8& ql,
                                             f32x16& acc, f32x16& low) {
  low = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, low, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
  low = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, low, 0, 0, 0);
}

// a value the compiler cannot see through: without it the double -> float -> half roundings of the first pairs become one
// long emulated conversion each, and the addresses of the loads are kept, spilled, for the stores at the end
template <typename V>
__device__ __forceinline__ V opaque(V v) {
  asm volatile("" : "+v"(v));
  return v;
}

// orders the LDS accesses of a wave's lanes (the hardware keeps their order, the compiler has to)
__device__ __forceinline__ void wave_meet() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

template <typename T, bool MOM, int NT>
__global__ __launch_bounds__(512) void small_kernel(const Group gr, float mu, float one_minus_mu, int nesterov,
                                                    float eps, int steps, float decay, float rate) {
  extern __shared__ __attribute__((aligned(16))) unsigned words[];      // read four at a time
  __shared__ double red[16];
  const Mat q = gr.mat[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, col = lane & 31, half = lane >> 5;
  unsigned* own = words + w * WAVE_WORDS;
  unsigned* sq_t = words + 8 * WAVE_WORDS;
  unsigned* sq_b = sq_t + 64 * SQUARE_ROW;
  const bool tall = q.rows > q.cols;
  // element e of row tile x of column tile t: row i, column j, and its place in the caller's matrix (0 behind the edges,
  // so that every load can be issued without a branch: a branch would wait for each in turn)
  auto row_of = [&](int x, int e) { return x * 32 + (e & 3) + 8 * (e >> 2) + 4 * half; };
  const unsigned si = tall ? 1 : q.cols, sj = tall ? q.cols : 1;
  unsigned corner = 4 * half * si + (w * 32 + col) * sj;
  int below = q.m - 4 * half, right = q.n - w * 32 - col;      // rows and columns there are from the corner on
  auto inside = [&](int x, int e, int t) { return x * 32 + (e & 3) + 8 * (e >> 2) < below && t * 256 < right; };
  auto place = [&](int x, int e, int t) {
    const unsigned at = corner + (x * 32 + (e & 3) + 8 * (e >> 2)) * si + t * 256 * sj;
    return inside(x, e, t) ? at : 0u;
  };
  float u[NT][2][16];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) u[t][x][e] = El<T>::get(q.g, place(x, e, t));
  if (MOM) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float m[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) m[e] = q.mom[place(x, e, t)];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float g = u[t][x][e];
          m[e] = fmaf(one_minus_mu, g - m[e], m[e]);
          if (inside(x, e, t)) q.mom[place(x, e, t)] = m[e];
          u[t][x][e] = direction(g, m[e], mu, nesterov);
        }
      }
  }
  double ss = 0.0;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (!inside(x, e, t)) u[t][x][e] = 0.f;
        ss += (double)u[t][x][e] * (double)u[t][x][e];
      }
  ss = block_sum_d(ss, red);
  const double norm = sqrt(ss);
  const double size = norm > (double)eps ? norm : (norm != norm ? norm : (double)eps);
  double r = norm / size;
  int k0 = extra_scale(r);
  const double mul0 = ldexp(1.0 / size, NS_SCALE + k0);
  f16x8 xh[NT][4], xl[NT][4];
  auto keep = [&](int t, int x, int e, float v) {
    const _Float16 hi = (_Float16)v;
    xh[t][x * 2 + (e >> 3)][e & 7] = hi;
    xl[t][x * 2 + (e >> 3)][e & 7] = (_Float16)(v - (float)hi);
  };
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) keep(t, x, e, opaque((float)((double)u[t][x][e] * mul0)));

  for (int step = 0; step < steps; ++step) {
    r = fmin((double)NS_A * r, 1.2025);
    const int k1 = extra_scale(r);
    // T = X X^T + shift: tiles (0, 0), (1, 0), (1, 1)
    f32x16 acc[3], low[3];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[k][e] = low[k][e] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if ((t * 8 + w) * 32 >= q.n) break;                    // uniform in the wave: the tile holds padding only
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const _Float16 p[2] = {xh[t][x * 2 + (e >> 3)][e & 7], xl[t][x * 2 + (e >> 3)][e & 7]};
          unsigned v;
          __builtin_memcpy(&v, p, 4);
          own[row_of(x, e) * TURN_ROW + col] = v;
        }
      wave_meet();
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        f16x8 ph[2], pl[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint4* p = reinterpret_cast<const uint4*>(own + (x * 32 + col) * TURN_ROW + g * 16 + half * 8);
          from_pairs(p[0], p[1], ph[x], pl[x]);
        }
        pair_product(ph[0], pl[0], ph[0], pl[0], acc[0], low[0]);
        pair_product(ph[1], pl[1], ph[0], pl[0], acc[1], low[1]);
        pair_product(ph[1], pl[1], ph[1], pl[1], acc[2], low[2]);
      }
      wave_meet();
    }
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) own[(k * 16 + e) * 64 + lane] = __float_as_uint(acc[k][e] + low[k][e]);
    __syncthreads();
    const float smul = ldexpf(1.f, -NS_SCALE - 2 * k0);
#pragma unroll
    for (int n = 0; n < WAVE_WORDS / 512; ++n) {
      const int at = n * 512 + tid, k = at >> 10, e = (at >> 6) & 15;
      float v = 0.f;
#pragma unroll
      for (int o = 0; o < 8; ++o) v += __uint_as_float(words[o * WAVE_WORDS + at]);
      const int i = row_of(k ? 1 : 0, e), j = (k == 2 ? 32 : 0) + col;
      v *= smul;
      if (i == j) v += ldexpf(NS_SHIFT, NS_SCALE);
      const unsigned p = to_pair(v);
      sq_t[i * SQUARE_ROW + j] = p;
      if (k == 1) sq_t[j * SQUARE_ROW + i] = p;
    }
    __syncthreads();
    // B = c T T + rest: one 32 x 32 tile for each of four waves
    if (w < 4) {
      const int x = w >> 1, y = w & 1;
      f32x16 b, bl;
#pragma unroll
      for (int e = 0; e < 16; ++e) b[e] = bl[e] = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f16x8 ph, pl, qh, ql;
        const uint4* p = reinterpret_cast<const uint4*>(sq_t + (x * 32 + col) * SQUARE_ROW + g * 16 + half * 8);
        const uint4* t = reinterpret_cast<const uint4*>(sq_t + (y * 32 + col) * SQUARE_ROW + g * 16 + half * 8);
        from_pairs(p[0], p[1], ph, pl);
        from_pairs(t[0], t[1], qh, ql);
        pair_product(ph, pl, qh, ql, b, bl);
      }
      const float bmul = ldexpf(NS_C, -NS_SCALE);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = row_of(x, e), j = y * 32 + col;
        sq_b[i * SQUARE_ROW + j] = to_pair((b[e] + bl[e]) * bmul + (i == j ? ldexpf(NS_REST, NS_SCALE) : 0.f));
      }
    }
    __syncthreads();
    // X = B X
    const float xmul = ldexpf(1.f, k1 - k0 - NS_SCALE);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if ((t * 8 + w) * 32 >= q.n) break;
      f32x16 d[2], dl[2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) d[x][e] = dl[x][e] = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          f16x8 ph, pl;
          const uint4* p = reinterpret_cast<const uint4*>(sq_b + (x * 32 + col) * SQUARE_ROW + g * 16 + half * 4);
          from_pairs(p[0], p[2], ph, pl);                    // rows 4 h + 0..3 and 8 + 4 h + 0..3 of these sixteen
          pair_product(ph, pl, xh[t][g], xl[t][g], d[x], dl[x]);
        }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) keep(t, x, e, (d[x][e] + dl[x][e]) * xmul);
    }
    k0 = k1;
  }
  const float omul = ldexpf(1.f, -NS_SCALE - k0);
  corner = opaque(corner);
  below = opaque(below);
  right = opaque(right);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float* p = static_cast<float*>(q.out);
      float old[16];
      if (MOM) {
#pragma unroll
        for (int e = 0; e < 16; ++e) old[e] = p[place(x, e, t)];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int g = x * 2 + (e >> 3);
        const float v = ((float)xh[t][g][e & 7] + (float)xl[t][g][e & 7]) * omul;
        if (!inside(x, e, t)) continue;
        if (MOM)
          p[place(x, e, t)] = fmaf(old[e], decay, -rate * q.adjust * v);
        else
          El<T>::put(q.out, place(x, e, t), v);
      }
    }
}

// ---- host side
constexpr int MAX_SIDE = 1 << 20;
constexpr long MAX_VALUES = 1l << 31;

int check_sizes(const int* rows, const int* cols, int count) {
  if (!rows || !cols || count < 1) return MMSA_ERR_ARG;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 1 || cols[i] < 1) return MMSA_ERR_ARG;
    if (rows[i] > MAX_SIDE || cols[i] > MAX_SIDE || (long)rows[i] * cols[i] > MAX_VALUES) return MMSA_ERR_LIMIT;
  }
  return MMSA_OK;
}

// How many of a list's next matrices share one set of launches: as many as their descriptors fit, up to a scratch of 1 GiB
// (in the largest padding).  That is four rounds of 256 x 256 tiles on every compute unit, beyond which company gains
// nothing (a single 4096 x 14336 matrix has 896 tiles); 24 of those together would ask for 20 GB.
constexpr long SET_BYTES = 1l << 30;
int set_of(const int* rows, const int* cols, int left) {
  long bytes = 0;
  int n = 0;
  for (; n < left && n < GROUP; ++n) {
    const int m = rows[n] < cols[n] ? rows[n] : cols[n], k = rows[n] < cols[n] ? cols[n] : rows[n];
    Mat q;
    q.mp = (m + 255) & ~255;
    q.np = (k + 255) & ~255;
    bytes += mat_bytes(q);
    if (n && bytes > SET_BYTES) break;
  }
  return n;
}

struct Plan {
  int bt[3];       // tile of the T, B and X products
  int from[GROUP];   // which of the caller's matrices each one is
  int blocks[PH_COUNT];
  long bytes;
};

long tri(long t) { return t * (t + 1) / 2; }

// What a phase costs in microseconds with BT x BT tiles, from measurements (squares of 256 to 4096 values): a block
// costs `start` plus `unit` per 32 values of K where it has a compute unit to itself and `full` where the chip is full
// (32 and 64: two blocks share a unit).  Larger tiles read less per product, so they win once they fill the chip.
struct TileCost {
  int bt, slots;
  float start, unit, full;
};
constexpr TileCost COST[4] = {
    {32, 512, 4.2f, 0.13f, 0.32f}, {64, 512, 4.0f, 0.27f, 0.54f}, {128, 256, 7.4f, 0.49f, 0.77f}, {256, 256, 9.6f, 2.25f, 2.25f}};

// blocks: how many, their K steps in all, the longest and the shortest of them
float phase_cost(const TileCost& c, long blocks, long steps, long longest, long shortest) {
  const float unit = blocks <= 256 ? c.unit + (c.full - c.unit) * (c.bt <= 64 ? 0.f : blocks / 256.f) : c.full;
  float rounds;
  if (longest == shortest)
    rounds = (float)((blocks + c.slots - 1) / c.slots);
  else
    rounds = (float)steps / c.slots / longest + (blocks <= c.slots ? 0.f : 0.5f);
  if (rounds < 1.f) rounds = 1.f;
  return rounds * (c.start + unit * longest);
}

struct Dims {
  int m, n;
};

// Everything that follows from the sizes alone: order (long K first, so that no long block starts last), padding, tiles,
// splits of K, the blocks of every launch and the scratch.
void make_plan(const int* rows, const int* cols, Group* gr, Plan* pl) {
  const int n = gr->count;
  Dims d[GROUP];
  for (int i = 0; i < n; ++i) {
    pl->from[i] = i;
    d[i].m = rows[i] < cols[i] ? rows[i] : cols[i];
    d[i].n = rows[i] < cols[i] ? cols[i] : rows[i];
  }
  for (int i = 1; i < n; ++i)
    for (int j = i; j > 0 && d[pl->from[j]].n > d[pl->from[j - 1]].n; --j) {
      const int t = pl->from[j];
      pl->from[j] = pl->from[j - 1];
      pl->from[j - 1] = t;
    }
  // the general product decides the padding
  float best = 0.f;
  int pad = 0;
  for (const TileCost& c : COST) {
    if (c.bt == 32) continue;
    long blocks = 0, steps = 0, longest = 0, shortest = 1l << 40;
    for (int i = 0; i < n; ++i) {
      const long mt = mmsa_cdiv(d[i].m, c.bt), t = mt * mmsa_cdiv(d[i].n, c.bt), k = mt * c.bt / 32;
      blocks += t;
      steps += t * k;
      if (k > longest) longest = k;
      if (k < shortest) shortest = k;
    }
    const float us = phase_cost(c, blocks, steps, longest, shortest);
    if (!pad || us < best) best = us, pad = c.bt;
  }
  int parts = 0;
  for (int i = 0; i < n; ++i) {
    Mat& q = gr->mat[i];
    q.rows = rows[pl->from[i]];
    q.cols = cols[pl->from[i]];
    q.m = d[pl->from[i]].m;
    q.n = d[pl->from[i]].n;
    q.mp = (q.m + pad - 1) / pad * pad;
    q.np = (q.n + pad - 1) / pad * pad;
    q.part0 = parts;
    // at most 512 partial sums: every block of the next kernel adds all of them up
    const long values = (long)q.rows * q.cols;
    q.chunk = (int)((values + 511) / 512 + 3) & ~3;
    if (q.chunk < 4096) q.chunk = 4096;
    q.nparts = mmsa_cdiv(values, q.chunk);
    parts += q.nparts;
  }
  pl->bt[TO_X] = pad;
  // The symmetric products: tile and share of K a block takes.  Partial tiles cost their way through memory and a
  // second launch.
  for (int ph = TO_T; ph <= TO_B; ++ph) {
    float least = 0.f;
    long share = 0;
    pl->bt[ph] = 0;
    for (const TileCost& c : COST) {
      if (c.bt > pad || c.bt == 256) break;       // errors of T count most: tiles with two accumulators only
      long work = 0, most = 0;
      for (int i = 0; i < n; ++i) {
        const long k = (ph == TO_T ? gr->mat[i].np : gr->mat[i].mp) / 32;
        work += tri(gr->mat[i].mp / c.bt) * k;
        if (k > most) most = k;
      }
      for (int rounds = 0; rounds <= 4; ++rounds) {       // 0: whole
        long kper = most;
        if (rounds) {
          kper = (work / (rounds * c.slots) + 2) & ~1l;
          if (kper < 4) kper = 4;
          if (kper >= most) continue;
        }
        long blocks = 0, longest = 0, shortest = 1l << 40, parted = 0, parts = 0;
        for (int i = 0; i < n; ++i) {
          const long k = (ph == TO_T ? gr->mat[i].np : gr->mat[i].mp) / 32, sp = (k + kper - 1) / kper;
          const long each = (k + sp - 1) / sp, t = tri(gr->mat[i].mp / c.bt) * sp;
          blocks += t;
          if (sp > 1) parted += t;
          if (sp > parts) parts = sp;
          if (each > longest) longest = each;
          if (each < shortest) shortest = each;
        }
        float us = phase_cost(c, blocks, work, longest, shortest);
        if (parted) us += 5.f + 0.04f * parts + (float)parted * c.bt * c.bt * 8 / 3e6f;
        if (!pl->bt[ph] || us < least) least = us, pl->bt[ph] = c.bt, share = kper;
      }
    }
    for (int i = 0; i < n; ++i) {
      Mat& q = gr->mat[i];
      const long k = (ph == TO_T ? q.np : q.mp) / 32, sp = (k + share - 1) / share;
      const long each = (k / 2 + sp - 1) / sp * 2;            // an even number of steps
      q.nsplit[ph] = (int)((k + each - 1) / each);            // no block without a step
    }
  }
  int total[PH_COUNT] = {0};
  long bytes = (sizeof(Group) + 127) / 128 * 128 + (8l * parts + 127) / 128 * 128;
  for (int i = 0; i < n; ++i) {
    Mat& q = gr->mat[i];
    q.ws_off = bytes;
    long part_floats = 0;
    for (int p = 0; p < PH_COUNT; ++p) gr->first[p][i] = total[p];
    total[PH_SUMSQ] += q.nparts;
    total[PH_SPLIT] += (q.mp / 64) * (q.np / 64);
    for (int ph = TO_T; ph <= TO_B; ++ph) {
      const int bt = pl->bt[ph];
      const long t = tri(q.mp / bt);
      total[PH_PRODUCT + ph] += (int)(t * q.nsplit[ph]);
      if (q.nsplit[ph] > 1) {
        total[PH_JOIN + ph] += (int)(t * (bt * bt / (many_parts(q.nsplit[ph]) ? 256 : 1024)));
        const long f = t * q.nsplit[ph] * bt * bt;
        if (f > part_floats) part_floats = f;
      }
    }
    total[PH_PRODUCT + TO_X] += (q.mp / pad) * (q.np / pad);
    bytes += mat_bytes(q) + 4 * part_floats;
  }
  for (int ph = 0; ph < 3; ++ph) {
    gr->even[ph] = 1;
    for (int i = 1; i < n; ++i) {
      const Mat &q = gr->mat[i], &o = gr->mat[0];
      if ((ph == TO_T ? q.np != o.np : q.mp != o.mp) || (ph < TO_X && q.nsplit[ph] != o.nsplit[ph])) gr->even[ph] = 0;
    }
  }
  for (int p = 0; p < PH_COUNT; ++p) pl->blocks[p] = total[p];
  pl->bytes = bytes;
}

struct Step {
  float mu, one_minus_mu;
  int nesterov;
  float eps, decay, rate;
  int steps;
};

template <typename T, int MODE>
void launch_product(const Plan& pl, const Group& gr, const Group* dev, int step, const Step& st, hipStream_t s) {
  constexpr int PHASE = MODE < TO_X ? MODE : TO_X;
  const dim3 grid(pl.blocks[PH_PRODUCT + PHASE]);
  if constexpr (MODE >= TO_X) {
    if (pl.bt[PHASE] == 256) {
      hipLaunchKernelGGL((product_kernel<T, 256, MODE>), grid, dim3(256), 0, s, dev, gr.count, gr.even[PHASE], step,
                       step & 1, st.decay, st.rate);
      return;
    }
  }
  if constexpr (MODE < TO_X) {
    if (pl.bt[PHASE] == 32) {
      hipLaunchKernelGGL((narrow_kernel<MODE>), grid, dim3(256), 0, s, dev, gr.count, gr.even[PHASE], step);
      return;
    }
  }
  if (pl.bt[PHASE] == 128)
    hipLaunchKernelGGL((product_kernel<T, 128, MODE>), grid, dim3(256), 0, s, dev, gr.count, gr.even[PHASE], step,
                       step & 1, st.decay, st.rate);
  else
    hipLaunchKernelGGL((product_kernel<T, 64, MODE>), grid, dim3(256), 0, s, dev, gr.count, gr.even[PHASE], step,
                       step & 1, st.decay, st.rate);
}
template <int MODE>
void launch_join(const Plan& pl, const Group& gr, const Group* dev, int step, hipStream_t s) {
  const int blocks = pl.blocks[PH_JOIN + MODE];
  if (!blocks) return;
  if (pl.bt[MODE] == 128)
    hipLaunchKernelGGL((join_kernel<128, MODE>), dim3(blocks), dim3(256), 0, s, dev, gr.count, step);
  else if (pl.bt[MODE] == 32)
    hipLaunchKernelGGL((join_kernel<32, MODE>), dim3(blocks), dim3(256), 0, s, dev, gr.count, step);
  else
    hipLaunchKernelGGL((join_kernel<64, MODE>), dim3(blocks), dim3(256), 0, s, dev, gr.count, step);
}

// raising a kernel's LDS limit belongs to the device that is current
template <auto kernel>
int allow_lds(size_t bytes) {
  static PerDeviceOnce once;
  if (once.pending()) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)bytes) != hipSuccess)
      return MMSA_ERR_LAUNCH;
    once.done();
  }
  return MMSA_OK;
}

// Which lists the kernel for small matrices takes, from both sides measured (one matrix, microseconds): 64 x 256 values
// 29 against 87 for 65 x 256 in the general launches, 64 x 512 44 against 95, 64 x 768 85 against 104.  An optimiser step
// holds the momentum beside the matrix: 64 x 512 57 against 96, but 64 x 576 103 against 98.
bool all_small(const int* rows, const int* cols, int count, int widest, int* longest) {
  *longest = 0;
  for (int i = 0; i < count; ++i) {
    const int m = rows[i] < cols[i] ? rows[i] : cols[i], n = rows[i] < cols[i] ? cols[i] : rows[i];
    if (m > SMALL_M || n > widest) return false;
    if (n > *longest) *longest = n;
  }
  return true;
}

template <typename T, bool MOM, int NT>
int launch_small(const Group& gr, const Step& st, hipStream_t s) {
  constexpr size_t lds = 4 * (8 * WAVE_WORDS + 2 * 64 * SQUARE_ROW);
  if (int rc = allow_lds<small_kernel<T, MOM, NT>>(lds)) return rc;
  hipLaunchKernelGGL((small_kernel<T, MOM, NT>), dim3(gr.count), dim3(512), lds, s, gr, st.mu, st.one_minus_mu,
                     st.nesterov, st.eps, st.steps, st.decay, st.rate);
  return mmsa_launch_status();
}

template <typename T, bool MOM>
int run_all(const void* const* src, void* const* dst, void* const* mom, const int* rows, const int* cols, int count,
            const Step& st, void* scratch, hipStream_t s) {
  for (int i0 = 0, n; i0 < count; i0 += n) {
    n = set_of(rows + i0, cols + i0, count - i0);
    Group gr;
    memset(&gr, 0, sizeof(gr));
    gr.count = n;
    Plan pl;
    make_plan(rows + i0, cols + i0, &gr, &pl);
    constexpr int NT_MOST = MOM ? 2 : 3;
    int longest;
    const bool small = all_small(rows + i0, cols + i0, gr.count, 256 * NT_MOST, &longest);
    for (int i = 0; i < gr.count; ++i) {
      Mat& q = gr.mat[i];
      const int at = i0 + pl.from[i];
      q.g = src[at];
      q.out = dst[at];
      q.mom = mom ? static_cast<float*>(mom[at]) : nullptr;
      q.ws = static_cast<char*>(scratch) + q.ws_off;
      q.adjust = q.rows > q.cols ? sqrtf((float)q.rows / (float)q.cols) : 1.f;
    }
    if (small) {
      const int rc = longest <= 256   ? launch_small<T, MOM, 1>(gr, st, s)
                     : longest <= 512 ? launch_small<T, MOM, 2>(gr, st, s)
                                      : launch_small<T, MOM, NT_MOST>(gr, st, s);
      if (rc) return rc;
      continue;
    }
    Group* dev = static_cast<Group*>(scratch);
    double* parts = reinterpret_cast<double*>(static_cast<char*>(scratch) + (sizeof(Group) + 127) / 128 * 128);
    hipLaunchKernelGGL((momentum_sumsq_kernel<T, MOM>), dim3(pl.blocks[PH_SUMSQ]), dim3(256), 0, s, gr, st.mu,
                       st.one_minus_mu, st.nesterov, parts, dev);
    hipLaunchKernelGGL((split_kernel<T, MOM>), dim3(pl.blocks[PH_SPLIT]), dim3(256), 0, s, dev, gr.count, st.mu, st.nesterov,
                       st.eps, st.steps, parts);
    for (int t = 0; t < st.steps; ++t) {
      launch_product<float, TO_T>(pl, gr, dev, t, st, s);
      launch_join<TO_T>(pl, gr, dev, t, s);
      launch_product<float, TO_B>(pl, gr, dev, t, st, s);
      launch_join<TO_B>(pl, gr, dev, t, s);
      if (t + 1 < st.steps)
        launch_product<float, TO_X>(pl, gr, dev, t, st, s);
      else
        launch_product<T, MOM ? TO_PARAM : TO_OUT>(pl, gr, dev, t, st, s);
    }
    if (int rc = mmsa_launch_status()) return rc;
  }
  return MMSA_OK;
}

bool pointers_ok(const void* const* p, int count) {
  if (!p) return false;
  for (int i = 0; i < count; ++i)
    if (!p[i]) return false;
  return true;
}

}  // namespace

// Bytes of scratch the two calls below need for these matrices (128-byte aligned).
MMSA_EXPORT long mmsa_orthogonalize_scratch_bytes(const int* rows_host, const int* cols_host, int count) {
  if (int rc = check_sizes(rows_host, cols_host, count)) return rc;
  long most = 0;
  for (int i0 = 0, n; i0 < count; i0 += n) {
    n = set_of(rows_host + i0, cols_host + i0, count - i0);
    Group gr;
    gr.count = n;
    Plan pl;
    make_plan(rows_host + i0, cols_host + i0, &gr, &pl);
    if (pl.bytes > most) most = pl.bytes;
  }
  return most;
}

MMSA_EXPORT int mmsa_orthogonalize(const void* const* src_host, void* const* dst_host, const int* rows_host,
                                   const int* cols_host, int count, int dtype, int steps, float eps, void* scratch,
                                   void* stream) {
  if (int rc = check_sizes(rows_host, cols_host, count)) return rc;
  MMSA_REQUIRE(pointers_ok(src_host, count) && pointers_ok(dst_host, count) && scratch);
  MMSA_REQUIRE(((unsigned long long)scratch & 127) == 0 && steps >= 1 && steps <= MAX_STEPS && eps > 0.f);
  const Step st{0.f, 1.f, 0, eps, 0.f, 0.f, steps};
  hipStream_t s = mmsa_stream(stream);
  if (dtype == 0) return run_all<float, false>(src_host, dst_host, nullptr, rows_host, cols_host, count, st, scratch, s);
  if (dtype == 1)
    return run_all<__hip_bfloat16, false>(src_host, dst_host, nullptr, rows_host, cols_host, count, st, scratch, s);
  if (dtype == 2)
    return run_all<_Float16, false>(src_host, dst_host, nullptr, rows_host, cols_host, count, st, scratch, s);
  return MMSA_ERR_ARG;
}

MMSA_EXPORT int mmsa_muon_step(void* const* params_host, const void* const* grads_host, void* const* momentum_host,
                               const int* rows_host, const int* cols_host, int count, double lr, double weight_decay,
                               double momentum, int nesterov, int steps, float eps, void* scratch, void* stream) {
  if (int rc = check_sizes(rows_host, cols_host, count)) return rc;
  MMSA_REQUIRE(pointers_ok(params_host, count) && pointers_ok(grads_host, count) && pointers_ok(momentum_host, count));
  MMSA_REQUIRE(scratch && ((unsigned long long)scratch & 127) == 0 && steps >= 1 && steps <= MAX_STEPS && eps > 0.f);
  const Step st{(float)momentum, (float)(1.0 - momentum), nesterov, eps, (float)(1.0 - lr * weight_decay), (float)lr,
                steps};
  return run_all<float, true>(grads_host, params_host, momentum_host, rows_host, cols_host, count, st, scratch,
                              mmsa_stream(stream));
}
