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
// which keeps 2^-24 relative (fp32's own half unit) down to 2^-39 absolute, and each product is three fp16 matrix
// products hi hi + hi lo + lo hi into one fp32 accumulator; lo lo is below 2^-24 relative and left out.  That is fp32
// accuracy at a third of the fp16 matrix rate (about 2.5 PFLOP/s) instead of the fp32 matrix rate (157 TFLOP/s).
// A matrix whose norm is below eps enters with entries far below 1: its X is held at a larger scale 2^(14 + k), k from
// the norm (the polynomial grows it by at most a per step, so k shrinks from step to step by the same bound).
//
// Layout.  A padded matrix [rows][K] of pairs is stored as [row][K / 32][hi 32 | lo 32] fp16: 32 values of a row are
// one 128-byte line holding both halves, which is what a K step of the products reads.  All products are row times row
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
constexpr int GROUP = 24;              // matrices of one launch (their descriptors travel as kernel arguments)
constexpr int CHUNK = 16384;           // values of one partial sum of squares

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
  int part0, nparts;    // its partial sums of squares
  int nsplit[2];        // blocks that share the K range of a tile of T / B
  float adjust;         // max(1, rows / cols)^1/2
  int pad_;
};
// The descriptors of one set of launches: an argument of the first kernel, which leaves them at the start of the
// scratch for the others (an argument of this size costs the host a few microseconds per launch).
struct Group {
  Mat mat[GROUP];
  int first[PH_COUNT][GROUP];   // first block of every matrix in each kind of launch
  int count, pad_;
};
static_assert(sizeof(Group) < 4096 - 256, "kernel arguments are limited to 4 KiB");

// scratch of one matrix: X [mp][np], X^T [np][mp] twice (read and written in turn), T and B [mp][mp], k per step, the
// partial tiles of a split product
__host__ __device__ inline long xbytes(const Mat& q) { return 4l * q.mp * q.np; }
__host__ __device__ inline long sbytes(const Mat& q) { return 4l * q.mp * q.mp; }
__device__ __forceinline__ char* ws_x(const Mat& q) { return q.ws; }
__device__ __forceinline__ char* ws_xt(const Mat& q, int which) { return q.ws + (1 + which) * xbytes(q); }
__device__ __forceinline__ char* ws_t(const Mat& q) { return q.ws + 3 * xbytes(q); }
__device__ __forceinline__ char* ws_b(const Mat& q) { return q.ws + 3 * xbytes(q) + sbytes(q); }
__device__ __forceinline__ int* ws_k(const Mat& q) { return reinterpret_cast<int*>(q.ws + 3 * xbytes(q) + 2 * sbytes(q)); }
__device__ __forceinline__ float* ws_part(const Mat& q) {
  return reinterpret_cast<float*>(q.ws + 3 * xbytes(q) + 2 * sbytes(q) + 128);
}

// which matrix a block works on: the last one whose first block is not behind it (all lanes of a wave call it)
__device__ __forceinline__ int find_mat(const int* first, int count, int block) {
  const int lane = threadIdx.x & 63;
  const bool at_or_behind = lane < count && first[lane < count ? lane : 0] <= block;
  // matrices without a block in this launch share their first block with the next one that has some
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(at_or_behind)) - 1);
}

// ---- element types
template <typename T> struct El;
template <> struct El<float> {
  static __device__ __forceinline__ float get(const void* p, long i) { return static_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ void put(void* p, long i, float v) { static_cast<float*>(p)[i] = v; }
};
template <> struct El<__hip_bfloat16> {
  static __device__ __forceinline__ float get(const void* p, long i) {
    return __uint_as_float((unsigned)static_cast<const unsigned short*>(p)[i] << 16);
  }
  static __device__ __forceinline__ void put(void* p, long i, float v) {
    static_cast<__hip_bfloat16*>(p)[i] = __float2bfloat16(v);
  }
};
template <> struct El<_Float16> {
  static __device__ __forceinline__ float get(const void* p, long i) {
    return (float)static_cast<const _Float16*>(p)[i];
  }
  static __device__ __forceinline__ void put(void* p, long i, float v) { static_cast<_Float16*>(p)[i] = (_Float16)v; }
};

__device__ __forceinline__ float direction(float g, float mom, float mu, int nesterov) {
  return nesterov ? fmaf(mu, mom - g, g) : mom;
}

// momentum update (MOM) and the sum of squares of u, one block per CHUNK values
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
  const long lo = (long)c * CHUNK, total = (long)q.rows * q.cols;
  const long hi = lo + CHUNK < total ? lo + CHUNK : total;
  double ss = 0.0;
  for (long j = lo + threadIdx.x; j < hi; j += 256) {
    float u = El<T>::get(q.g, j);
    if (MOM) {
      const float g = u;
      const float m = fmaf(one_minus_mu, g - q.mom[j], q.mom[j]);
      q.mom[j] = m;
      u = direction(g, m, mu, nesterov);
    }
    ss += (double)u * (double)u;
  }
  ss = block_sum_d(ss, red);
  if (threadIdx.x == 0) parts[q.part0 + c] = ss;
}

__device__ __forceinline__ void put_pair(char* base, long row, long col, long K, float v) {
  const _Float16 hi = (_Float16)v;
  _Float16* p = reinterpret_cast<_Float16*>(base) + row * 2 * K + (col >> 5) * 64 + (col & 31);
  p[0] = hi;
  p[32] = (_Float16)(v - (float)hi);
}

// how far X's scale exceeds 2^NS_SCALE for a bound r on its norm
__device__ __forceinline__ int extra_scale(double r) {
  if (!(r > 0.0) || r >= 1.0) return 0;
  return min(400, max(0, (int)floor(-log2(r))));
}

// normalises u and writes X and X^T as pairs, 64 x 64 values of u's padded extent per block
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void split_kernel(const Group* __restrict__ grp, float mu, int nesterov, float eps,
                                                    int steps, const double* __restrict__ parts) {
  __shared__ double red[16];
  __shared__ float tile[64][65];
  const Group& gr = *grp;
  const int i = find_mat(gr.first[PH_SPLIT], gr.count, blockIdx.x);
  const Mat& q = gr.mat[i];
  const int b = blockIdx.x - gr.first[PH_SPLIT][i];
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
  const bool tall = q.rows > q.cols;
  const int pr = tall ? q.np : q.mp, pc = tall ? q.mp : q.np;      // padded extent in u's own orientation
  const int nct = pc / 64;
  const long r0 = (long)(b / nct) * 64, c0 = (long)(b % nct) * 64;
  char* rowm = tall ? ws_xt(q, 0) : ws_x(q);                       // [pr][pc]
  char* colm = tall ? ws_x(q) : ws_xt(q, 0);                       // [pc][pr]
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int rr = ty; rr < 64; rr += 4) {
    const long row = r0 + rr, col = c0 + tx;
    float v = 0.f;
    if (row < q.rows && col < q.cols) {
      const long at = row * q.cols + col;
      float u = El<T>::get(q.g, at);
      if (MOM) u = direction(u, q.mom[at], mu, nesterov);
      v = (float)((double)u * mul);
    }
    tile[rr][tx] = v;
    put_pair(rowm, row, col, pc, v);
  }
  __syncthreads();
  for (int cc = ty; cc < 64; cc += 4) put_pair(colm, c0 + cc, r0 + tx, pr, tile[tx][cc]);
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

// D = P Q^T over K for one BT x BT tile, four waves as 2 x 2, both operands staged through LDS in K steps of 32 values
// (128-byte rows, their 16-byte units XORed with the row so that the fragment reads spread over the banks).
// T and B are symmetric: only tiles on and below the diagonal are computed, the others are written as their mirror
// image.  Where a phase has few tiles and a long K, `kper` steps of K go to one block each and the partial results
// meet in join_kernel.
template <typename T, int BT, int MODE>
__global__ __launch_bounds__(256) void product_kernel(const Group* __restrict__ grp, int step, int which, float decay,
                                                      float rate) {
  constexpr int WT = BT / 64;                 // 32 x 32 tiles a wave has per direction
  constexpr int OPER = BT * 128;              // bytes of one operand's stage
  constexpr int OUTROW = BT * 4 + 16;         // an output row of pairs in LDS, padded against bank conflicts
  __shared__ __attribute__((aligned(128))) char lds[4 * OPER > BT * OUTROW ? 4 * OPER : BT * OUTROW];
  const Group& gr = *grp;
  constexpr int PHASE = MODE < TO_X ? MODE : TO_X;
  const int mi = find_mat(gr.first[PH_PRODUCT + PHASE], gr.count, blockIdx.x);
  const Mat& q = gr.mat[mi];
  int b = blockIdx.x - gr.first[PH_PRODUCT + PHASE][mi];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int K = MODE == TO_T ? q.np : q.mp;
  int ti, tj, k_lo = 0, nk = K / 32, part = 0, nsplit = 1, tile = 0;
  if (MODE <= TO_B) {
    nsplit = q.nsplit[PHASE];
    tile = b / nsplit;
    part = b % nsplit;
    lower_tile(tile, ti, tj);
    const int kper = (nk + nsplit - 1) / nsplit;
    k_lo = part * kper;
    nk = nk - k_lo < kper ? nk - k_lo : kper;
  } else {
    const int nt = q.np / BT;
    ti = b / nt;
    tj = b % nt;
  }
  const char* P = MODE == TO_T ? ws_x(q) : MODE == TO_B ? ws_t(q) : ws_b(q);
  const char* Q = MODE == TO_T ? ws_x(q) : MODE == TO_B ? ws_t(q) : ws_xt(q, which);
  const long pitch = 4l * K;
  // staging: a wave's load fills eight rows of 128 bytes
  const int lrow = lane >> 3, lunit = (lane & 7) ^ lrow;
  const char* ps = P + ((long)ti * BT + w * 8 + lrow) * pitch + lunit * 16 + k_lo * 128l;
  const char* qs = Q + ((long)tj * BT + w * 8 + lrow) * pitch + lunit * 16 + k_lo * 128l;
  auto stage = [&](int buf, int kc) {
#pragma unroll
    for (int j = 0; j < BT / 32; ++j) {
      load_lds16(ps + j * 32 * pitch + (long)kc * 128, lds + (buf * 2 + 0) * OPER + (j * 32 + w * 8) * 128);
      load_lds16(qs + j * 32 * pitch + (long)kc * 128, lds + (buf * 2 + 1) * OPER + (j * 32 + w * 8) * 128);
    }
  };
  f32x16 acc[WT][WT];
#pragma unroll
  for (int x = 0; x < WT; ++x)
#pragma unroll
    for (int y = 0; y < WT; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  const int wi = w >> 1, wj = w & 1;
  const int fr = lane & 31, half = lane >> 5;
  if (nk > 0) stage(0, 0);
  for (int kc = 0; kc < nk; ++kc) {
    __syncthreads();
    if (kc + 1 < nk) stage((kc + 1) & 1, kc + 1);
    const char* lp = lds + (kc & 1) * 2 * OPER;
    const char* lq = lp + OPER;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f16x8 ph[WT], pl[WT], qh[WT], ql[WT];
#pragma unroll
      for (int x = 0; x < WT; ++x) {
        const int rp = wi * (BT / 2) + x * 32 + fr, rq = wj * (BT / 2) + x * 32 + fr;
        const int u = s * 2 + half;
        ph[x] = *reinterpret_cast<const f16x8*>(lp + rp * 128 + ((u ^ (rp & 7)) * 16));
        pl[x] = *reinterpret_cast<const f16x8*>(lp + rp * 128 + (((u + 4) ^ (rp & 7)) * 16));
        qh[x] = *reinterpret_cast<const f16x8*>(lq + rq * 128 + ((u ^ (rq & 7)) * 16));
        ql[x] = *reinterpret_cast<const f16x8*>(lq + rq * 128 + (((u + 4) ^ (rq & 7)) * 16));
      }
#pragma unroll
      for (int x = 0; x < WT; ++x)
#pragma unroll
        for (int y = 0; y < WT; ++y) {
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[x], qh[y], acc[x][y], 0, 0, 0);
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[x], ql[y], acc[x][y], 0, 0, 0);
          acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[x], qh[y], acc[x][y], 0, 0, 0);
        }
    }
  }
  // register e of a wave's tile (x, y): row (e & 3) + 8 (e >> 2) + 4 half, column fr
  if (MODE <= TO_B && nsplit > 1) {
    float* o = ws_part(q) + ((long)tile * nsplit + part) * (BT * BT) + tid;
#pragma unroll
    for (int x = 0; x < WT; ++x)
#pragma unroll
      for (int y = 0; y < WT; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[((x * WT + y) * 16 + e) * 256] = acc[x][y][e];
    return;
  }
  const float mul = result_scale<MODE>(q, step);
  const int i0 = wi * (BT / 2) + 4 * half, j0 = wj * (BT / 2) + fr;
  if (MODE >= TO_OUT) {
    const bool tall = q.rows > q.cols;
#pragma unroll
    for (int x = 0; x < WT; ++x)
#pragma unroll
      for (int y = 0; y < WT; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const long i = (long)ti * BT + i0 + x * 32 + (e & 3) + 8 * (e >> 2), j = (long)tj * BT + j0 + y * 32;
          if (i >= q.m || j >= q.n) continue;
          const float v = acc[x][y][e] * mul;
          const long at = tall ? j * q.cols + i : i * q.cols + j;
          if (MODE == TO_OUT) {
            El<T>::put(q.out, at, v);
          } else {
            float* p = static_cast<float*>(q.out);
            p[at] = fmaf(p[at], decay, -rate * q.adjust * v);
          }
        }
    return;
  }
  // the tile and its transpose leave through LDS as rows of pairs
  const bool diag = MODE <= TO_B && ti == tj;
#pragma unroll
  for (int x = 0; x < WT; ++x)
#pragma unroll
    for (int y = 0; y < WT; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float v = acc[x][y][e] * mul;
        if (diag && i0 + x * 32 + (e & 3) + 8 * (e >> 2) == j0 + y * 32) v += diagonal<MODE>();
        acc[x][y][e] = v;
      }
  char* direct = MODE == TO_T ? ws_t(q) : MODE == TO_B ? ws_b(q) : ws_x(q);
  char* mirror = MODE == TO_X ? ws_xt(q, which ^ 1) : direct;
  const long dpitch = 4l * (MODE == TO_X ? q.np : q.mp), mpitch = 4l * q.mp;
  auto copy_out = [&](char* dst, long dst_pitch) {
    for (int u = tid; u < BT * BT / 4; u += 256) {
      const int row = u / (BT / 4), unit = u % (BT / 4);
      *reinterpret_cast<uint4*>(dst + row * dst_pitch + unit * 16) =
          *reinterpret_cast<const uint4*>(lds + row * OUTROW + unit * 16);
    }
  };
  __syncthreads();
#pragma unroll
  for (int x = 0; x < WT; ++x)
#pragma unroll
    for (int y = 0; y < WT; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = i0 + x * 32 + (e & 3) + 8 * (e >> 2), j = j0 + y * 32;
        const float v = acc[x][y][e];
        const _Float16 hi = (_Float16)v;
        _Float16* o = reinterpret_cast<_Float16*>(lds + i * OUTROW + (j >> 5) * 128) + (j & 31);
        o[0] = hi;
        o[32] = (_Float16)(v - (float)hi);
      }
  __syncthreads();
  copy_out(direct + (long)ti * BT * dpitch + tj * (BT * 4l), dpitch);
  if (diag) return;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < WT; ++x)
#pragma unroll
    for (int y = 0; y < WT; ++y)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int i = i0 + x * 32 + 8 * g, j = j0 + y * 32;
        f16x4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = acc[x][y][g * 4 + r];
          hi[r] = (_Float16)v;
          lo[r] = (_Float16)(v - (float)hi[r]);
        }
        char* o = lds + j * OUTROW + (i >> 5) * 128 + (i & 31) * 2;
        *reinterpret_cast<f16x4*>(o) = hi;
        *reinterpret_cast<f16x4*>(o + 64) = lo;
      }
  __syncthreads();
  copy_out(mirror + (long)tj * BT * mpitch + ti * (BT * 4l), mpitch);
}

// sums the partial tiles of the matrices whose K was split, one value per thread in the product kernel's register order
template <int BT, int MODE>
__global__ __launch_bounds__(256) void join_kernel(const Group* __restrict__ grp, int step) {
  constexpr int WT = BT / 64, PER = BT * BT / 256;
  const Group& gr = *grp;
  const int mi = find_mat(gr.first[PH_JOIN + MODE], gr.count, blockIdx.x);
  const Mat& q = gr.mat[mi];
  const int b = blockIdx.x - gr.first[PH_JOIN + MODE][mi];
  const int tile = b / PER, r = b % PER, tid = threadIdx.x;
  const int nsplit = q.nsplit[MODE];
  int ti, tj;
  lower_tile(tile, ti, tj);
  const float* p = ws_part(q) + (long)tile * nsplit * (BT * BT) + r * 256 + tid;
  float v = 0.f;
  for (int s = 0; s < nsplit; ++s) v += p[(long)s * (BT * BT)];
  v *= result_scale<MODE>(q, step);
  const int e = r & 15, x = (r >> 4) / WT, y = (r >> 4) % WT, lane = tid & 63, w = tid >> 6;
  const long i = (long)ti * BT + (w >> 1) * (BT / 2) + x * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
  const long j = (long)tj * BT + (w & 1) * (BT / 2) + y * 32 + (lane & 31);
  if (i == j) v += diagonal<MODE>();
  char* dst = MODE == TO_T ? ws_t(q) : ws_b(q);
  put_pair(dst, i, j, q.mp, v);
  if (ti != tj) put_pair(dst, j, i, q.mp, v);
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

struct Plan {
  int bt[3];       // tile of the T, B and X products
  int blocks[PH_COUNT];
  long bytes;
};

long tri(long t) { return t * (t + 1) / 2; }

// Everything that follows from the sizes alone: padding, tiles, splits, the blocks of every launch and the scratch.
// Tiles are 128 x 128 (a wave's 64 x 64 reads half as much LDS per product as 32 x 32) where a phase then still has
// ENOUGH tiles to occupy the chip, else 64 x 64; a phase with fewer blocks than that, or with one K much longer than
// the others', cuts K so that no block has more than its share of TARGET blocks.
constexpr int ENOUGH = 192, TARGET = 512, MIN_STEPS = 8;

void make_plan(const int* rows, const int* cols, Group* gr, Plan* pl) {
  const int n = gr->count;
  long x128 = 0;
  for (int i = 0; i < n; ++i)
    x128 += (long)mmsa_cdiv(rows[i], 128) * mmsa_cdiv(cols[i], 128);
  const int pad = x128 >= ENOUGH ? 128 : 64;
  int parts = 0;
  for (int i = 0; i < n; ++i) {
    Mat& q = gr->mat[i];
    q.rows = rows[i];
    q.cols = cols[i];
    q.m = rows[i] < cols[i] ? rows[i] : cols[i];
    q.n = rows[i] < cols[i] ? cols[i] : rows[i];
    q.mp = (q.m + pad - 1) / pad * pad;
    q.np = (q.n + pad - 1) / pad * pad;
    q.part0 = parts;
    q.nparts = mmsa_cdiv((long)rows[i] * cols[i], CHUNK);
    parts += q.nparts;
  }
  pl->bt[TO_X] = pad;
  for (int ph = TO_T; ph <= TO_B; ++ph) {
    long t128 = 0, work = 0, longest = 0, tiles = 0;
    for (int i = 0; i < n; ++i) t128 += tri(gr->mat[i].mp / 128);
    const int bt = pad == 128 && t128 >= ENOUGH ? 128 : 64;
    pl->bt[ph] = bt;
    for (int i = 0; i < n; ++i) {
      const Mat& q = gr->mat[i];
      const long t = tri(q.mp / bt), k = (ph == TO_T ? q.np : q.mp) / 32;
      tiles += t;
      work += t * k;
      if (k > longest) longest = k;
    }
    long kper = (work + TARGET - 1) / TARGET;
    if (kper < MIN_STEPS) kper = MIN_STEPS;
    const bool split = tiles < ENOUGH || longest > 2 * kper;
    for (int i = 0; i < n; ++i) {
      Mat& q = gr->mat[i];
      const long k = (ph == TO_T ? q.np : q.mp) / 32;
      int sp = split ? (int)((k + kper - 1) / kper) : 1;
      const int each = (int)((k + sp - 1) / sp);
      q.nsplit[ph] = (int)((k + each - 1) / each);       // no block without a step
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
        total[PH_JOIN + ph] += (int)(t * (bt * bt / 256));
        const long f = t * q.nsplit[ph] * bt * bt;
        if (f > part_floats) part_floats = f;
      }
    }
    total[PH_PRODUCT + TO_X] += (q.mp / pad) * (q.np / pad);
    bytes += 3 * xbytes(q) + 2 * sbytes(q) + 128 + 4 * part_floats;
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
void launch_product(const Plan& pl, const Group* dev, int step, const Step& st, hipStream_t s) {
  constexpr int PHASE = MODE < TO_X ? MODE : TO_X;
  const dim3 grid(pl.blocks[PH_PRODUCT + PHASE]), block(256);
  if (pl.bt[PHASE] == 128)
    hipLaunchKernelGGL((product_kernel<T, 128, MODE>), grid, block, 0, s, dev, step, step & 1, st.decay, st.rate);
  else
    hipLaunchKernelGGL((product_kernel<T, 64, MODE>), grid, block, 0, s, dev, step, step & 1, st.decay, st.rate);
}
template <int MODE>
void launch_join(const Plan& pl, const Group* dev, int step, hipStream_t s) {
  const int blocks = pl.blocks[PH_JOIN + MODE];
  if (!blocks) return;
  if (pl.bt[MODE] == 128)
    hipLaunchKernelGGL((join_kernel<128, MODE>), dim3(blocks), dim3(256), 0, s, dev, step);
  else
    hipLaunchKernelGGL((join_kernel<64, MODE>), dim3(blocks), dim3(256), 0, s, dev, step);
}

template <typename T, bool MOM>
int run_all(const void* const* src, void* const* dst, void* const* mom, const int* rows, const int* cols, int count,
            const Step& st, void* scratch, hipStream_t s) {
  for (int i0 = 0; i0 < count; i0 += GROUP) {
    Group gr;
    memset(&gr, 0, sizeof(gr));
    gr.count = count - i0 < GROUP ? count - i0 : GROUP;
    Plan pl;
    make_plan(rows + i0, cols + i0, &gr, &pl);
    for (int i = 0; i < gr.count; ++i) {
      Mat& q = gr.mat[i];
      q.g = src[i0 + i];
      q.out = dst[i0 + i];
      q.mom = mom ? static_cast<float*>(mom[i0 + i]) : nullptr;
      q.ws = static_cast<char*>(scratch) + q.ws_off;
      q.adjust = q.rows > q.cols ? sqrtf((float)q.rows / (float)q.cols) : 1.f;
    }
    Group* dev = static_cast<Group*>(scratch);
    double* parts = reinterpret_cast<double*>(static_cast<char*>(scratch) + (sizeof(Group) + 127) / 128 * 128);
    hipLaunchKernelGGL((momentum_sumsq_kernel<T, MOM>), dim3(pl.blocks[PH_SUMSQ]), dim3(256), 0, s, gr, st.mu,
                       st.one_minus_mu, st.nesterov, parts, dev);
    hipLaunchKernelGGL((split_kernel<T, MOM>), dim3(pl.blocks[PH_SPLIT]), dim3(256), 0, s, dev, st.mu, st.nesterov,
                       st.eps, st.steps, parts);
    for (int t = 0; t < st.steps; ++t) {
      launch_product<float, TO_T>(pl, dev, t, st, s);
      launch_join<TO_T>(pl, dev, t, s);
      launch_product<float, TO_B>(pl, dev, t, st, s);
      launch_join<TO_B>(pl, dev, t, s);
      if (t + 1 < st.steps)
        launch_product<float, TO_X>(pl, dev, t, st, s);
      else
        launch_product<T, MOM ? TO_PARAM : TO_OUT>(pl, dev, t, st, s);
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
  for (int i0 = 0; i0 < count; i0 += GROUP) {
    Group gr;
    gr.count = count - i0 < GROUP ? count - i0 : GROUP;
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
