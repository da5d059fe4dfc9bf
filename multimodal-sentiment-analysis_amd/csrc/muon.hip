// Orthogonalised updates of weight matrices (Newton-Schulz products) and the Muon optimiser step built on them.
//
//   X_0 = u / max(||u||_F, eps)          (u^T where u has more rows than columns: X is [m][n] with m <= n)
//   X <- (a I + b S + c S S) X,  S = X X^T,   `steps` times, (a, b, c) = (3.4445, -4.775, 2.0315)
// and for the optimiser   m <- m + (1 - mu)(g - m),  u = nesterov ? g + mu (m - g) : m,
//   p <- p (1 - lr wd) - lr max(1, rows / cols)^1/2 X_steps.
//
// Arithmetic.  x -> a x + b x^3 + c x^5 maps [0, 1.2025] into itself, so singular values, hence entries, of X never
// exceed 1.2025, those of S 1.446 and those of B = a I + b S + c S S 3.4445: every operand fits ONE fixed power-of-two
// scale of 2^14 in fp16, with no overflow for any input.  Each value is held as a pair hi = fp16(v), lo = fp16(v - hi),
// which keeps 2^-24 relative (fp32's own half unit) down to 2^-39 absolute, and each product is three fp16 matrix
// products hi hi + hi lo + lo hi into one fp32 accumulator; lo lo is below 2^-24 relative and left out.  That is fp32
// accuracy at a third of the fp16 matrix rate (about 2.5 PFLOP/s) instead of the fp32 matrix rate (157 TFLOP/s).
// A matrix whose norm is below eps enters with entries far below 1: its X is held at a larger scale 2^(14 + k), k from
// the norm (the polynomial grows it by at most a per step, so k shrinks from step to step by the same bound).
//
// Layout.  A padded matrix [rows][K] of pairs is stored as [row][K / 32][hi 32 | lo 32] fp16: 32 values of a row are
// one 128-byte line holding both halves, which is what a K step of the products reads.  All products are row times row
// (both operands K-contiguous): S = X X^T, S S (S is symmetric), and B X = B (X^T)^T, for which X^T is kept beside X.
// Padding rows and columns hold zeros and stay zero.
#include "mmsa_common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <string.h>

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float NS_A = 3.4445f, NS_B = -4.775f, NS_C = 2.0315f;
constexpr int NS_SCALE = 14;           // log2 of the fixed-point scale
constexpr int MAX_STEPS = 16;
constexpr int GROUP = 24;              // matrices of one launch (their descriptors travel as kernel arguments)
constexpr int CHUNK = 16384;           // values of one partial sum of squares

struct Mat {
  const void* g;        // gradient / input matrix, [rows][cols]
  void* out;            // orthogonalised matrix (same type as g) or the parameter (fp32), [rows][cols]
  float* mom;           // momentum buffer, or null
  char* ws;             // this matrix's part of the scratch
  int rows, cols;
  int m, n;             // the smaller and the larger of the two
  int mp, np;           // padded to the tile
  int part0, nparts;    // its partial sums of squares
  float adjust;         // max(1, rows / cols)^1/2
  int pad_;
};
struct Group {
  Mat mat[GROUP];
  int first[GROUP + 1];   // first block of every matrix in this launch
  int count;
};
static_assert(sizeof(Group) < 4096 - 256, "kernel arguments are limited to 4 KiB");

// scratch of one matrix: X [mp][np], X^T [np][mp] twice (read and written in turn), S and B [mp][mp], k per step
__host__ __device__ inline long xbytes(const Mat& q) { return 4l * q.mp * q.np; }
__host__ __device__ inline long sbytes(const Mat& q) { return 4l * q.mp * q.mp; }
__host__ __device__ inline long mat_bytes(const Mat& q) { return 3 * xbytes(q) + 2 * sbytes(q) + 128; }
__device__ __forceinline__ char* ws_x(const Mat& q) { return q.ws; }
__device__ __forceinline__ char* ws_xt(const Mat& q, int which) { return q.ws + (1 + which) * xbytes(q); }
__device__ __forceinline__ char* ws_s(const Mat& q) { return q.ws + 3 * xbytes(q); }
__device__ __forceinline__ char* ws_b(const Mat& q) { return q.ws + 3 * xbytes(q) + sbytes(q); }
__device__ __forceinline__ int* ws_k(const Mat& q) { return reinterpret_cast<int*>(q.ws + 3 * xbytes(q) + 2 * sbytes(q)); }

__device__ __forceinline__ int find_mat(const Group& gr, int block) {
  int i = 0;
  while (i + 1 < gr.count && block >= gr.first[i + 1]) ++i;
  return i;
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
                                                             double* __restrict__ parts) {
  __shared__ double red[16];
  const int i = find_mat(gr, blockIdx.x);
  const Mat& q = gr.mat[i];
  const int c = blockIdx.x - gr.first[i];
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
__global__ __launch_bounds__(256) void split_kernel(const Group gr, float mu, int nesterov, float eps, int steps,
                                                    const double* __restrict__ parts) {
  __shared__ double red[16];
  __shared__ float tile[64][65];
  const int i = find_mat(gr, blockIdx.x);
  const Mat& q = gr.mat[i];
  const int b = blockIdx.x - gr.first[i];
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
enum { TO_S = 0, TO_B = 1, TO_X = 2, TO_OUT = 3, TO_PARAM = 4 };

// 16 bytes per lane straight into LDS: lane l of the wave lands at lds + 16 l
__device__ __forceinline__ void load_lds16(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// D = P Q^T over K for one BT x BT tile, four waves as 2 x 2, both operands staged through LDS in K steps of 32 values
// (128-byte rows, their 16-byte units XORed with the row so that the fragment reads spread over the banks).
template <typename T, int BT, int MODE>
__global__ __launch_bounds__(256) void product_kernel(const Group gr, int step, int which, float decay, float rate) {
  constexpr int WT = BT / 64;                 // 32 x 32 tiles a wave has per direction
  constexpr int OPER = BT * 128;              // bytes of one operand's stage
  __shared__ __attribute__((aligned(128))) char lds[2][2][OPER];
  const int mi = find_mat(gr, blockIdx.x);
  const Mat& q = gr.mat[mi];
  int b = blockIdx.x - gr.first[mi];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int ti, tj;
  if (MODE <= TO_B) {                         // lower triangle of tiles: the result is symmetric
    ti = (int)((sqrtf(8.f * (float)b + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
    while (ti * (ti + 1) / 2 > b) --ti;
    tj = b - ti * (ti + 1) / 2;
  } else {
    const int nt = q.np / BT;
    ti = b / nt;
    tj = b % nt;
  }
  const char* P = MODE == TO_S ? ws_x(q) : MODE == TO_B ? ws_s(q) : ws_b(q);
  const char* Q = MODE == TO_S ? ws_x(q) : MODE == TO_B ? ws_s(q) : ws_xt(q, which);
  const int K = MODE == TO_S ? q.np : q.mp;
  const long pitch = 4l * K;
  // staging: a wave's load fills eight rows of 128 bytes
  const int lrow = lane >> 3, lunit = (lane & 7) ^ lrow;
  const char* ps = P + ((long)ti * BT + w * 8 + lrow) * pitch + lunit * 16;
  const char* qs = Q + ((long)tj * BT + w * 8 + lrow) * pitch + lunit * 16;
  auto stage = [&](int buf, int kc) {
#pragma unroll
    for (int j = 0; j < BT / 32; ++j) {
      load_lds16(ps + j * 32 * pitch + (long)kc * 128, &lds[buf][0][(j * 32 + w * 8) * 128]);
      load_lds16(qs + j * 32 * pitch + (long)kc * 128, &lds[buf][1][(j * 32 + w * 8) * 128]);
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
  const int nk = K / 32;
  stage(0, 0);
  for (int kc = 0; kc < nk; ++kc) {
    __syncthreads();
    if (kc + 1 < nk) stage((kc + 1) & 1, kc + 1);
    const char* lp = lds[kc & 1][0];
    const char* lq = lds[kc & 1][1];
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
  const int k0 = ws_k(q)[step], k1 = ws_k(q)[step + 1];
  const float xmul = MODE == TO_S   ? ldexpf(1.f, -NS_SCALE - 2 * k0)
                     : MODE == TO_B ? ldexpf(NS_C, -NS_SCALE)
                     : MODE == TO_X ? ldexpf(1.f, k1 - k0 - NS_SCALE)
                                    : ldexpf(1.f, -2 * NS_SCALE - k0);
  const bool tall = q.rows > q.cols;
  // register e of a tile: row (e & 3) + 8 (e >> 2) + 4 half, column fr
#pragma unroll
  for (int x = 0; x < WT; ++x)
#pragma unroll
    for (int y = 0; y < WT; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const long i = (long)ti * BT + wi * (BT / 2) + x * 32 + (e & 3) + 8 * (e >> 2) + 4 * half;
        const long j = (long)tj * BT + wj * (BT / 2) + y * 32 + fr;
        float v = acc[x][y][e] * xmul;
        if (MODE == TO_S) {
          put_pair(ws_s(q), i, j, q.mp, v);
          if (ti != tj) put_pair(ws_s(q), j, i, q.mp, v);
        } else if (MODE == TO_B) {
          const _Float16* sp = reinterpret_cast<const _Float16*>(ws_s(q)) + i * 2 * q.mp + (j >> 5) * 64 + (j & 31);
          v = fmaf(NS_B, (float)sp[0] + (float)sp[32], v);
          if (i == j) v += ldexpf(NS_A, NS_SCALE);
          put_pair(ws_b(q), i, j, q.mp, v);
          if (ti != tj) put_pair(ws_b(q), j, i, q.mp, v);
        } else if (MODE == TO_X) {
          put_pair(ws_x(q), i, j, q.np, v);
          put_pair(ws_xt(q, which ^ 1), j, i, q.mp, v);
        } else if (i < q.m && j < q.n) {
          const long at = tall ? j * q.cols + i : i * q.cols + j;
          if (MODE == TO_OUT) {
            El<T>::put(q.out, at, v);
          } else {
            float* p = static_cast<float*>(q.out);
            p[at] = fmaf(p[at], decay, -rate * q.adjust * v);
          }
        }
      }
}

// ---- host side
int tile_of(const int* rows, const int* cols, int count) {
  (void)rows; (void)cols; (void)count;
  return 64;
}

void shape_mat(Mat* q, int rows, int cols, int bt) {
  q->rows = rows;
  q->cols = cols;
  q->m = rows < cols ? rows : cols;
  q->n = rows < cols ? cols : rows;
  q->mp = (q->m + bt - 1) / bt * bt;
  q->np = (q->n + bt - 1) / bt * bt;
  q->nparts = mmsa_cdiv((long)rows * cols, CHUNK);
}

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

long scratch_bytes(const int* rows, const int* cols, int count) {
  long most = 0;
  for (int i0 = 0; i0 < count; i0 += GROUP) {
    const int n = count - i0 < GROUP ? count - i0 : GROUP;
    const int bt = tile_of(rows + i0, cols + i0, n);
    long bytes = 0, parts = 0;
    for (int i = 0; i < n; ++i) {
      Mat q;
      shape_mat(&q, rows[i0 + i], cols[i0 + i], bt);
      bytes += mat_bytes(q);
      parts += q.nparts;
    }
    bytes += 8 * parts + 256;
    if (bytes > most) most = bytes;
  }
  return most;
}

template <typename F>
int layout(Group* gr, F blocks_of) {
  int total = 0;
  for (int i = 0; i < gr->count; ++i) {
    gr->first[i] = total;
    total += blocks_of(gr->mat[i]);
  }
  gr->first[gr->count] = total;
  return total;
}

struct Step {
  int momentum;
  float mu, one_minus_mu;
  int nesterov;
  float eps, decay, rate;
  int steps;
};

template <typename T, bool MOM, int BT>
void launch_group(Group& gr, const Step& st, double* parts, hipStream_t s) {
  int blocks = layout(&gr, [](const Mat& q) { return q.nparts; });
  hipLaunchKernelGGL((momentum_sumsq_kernel<T, MOM>), dim3(blocks), dim3(256), 0, s, gr, st.mu, st.one_minus_mu,
                     st.nesterov, parts);
  blocks = layout(&gr, [](const Mat& q) { return (q.mp / 64) * (q.np / 64); });
  hipLaunchKernelGGL((split_kernel<T, MOM>), dim3(blocks), dim3(256), 0, s, gr, st.mu, st.nesterov, st.eps, st.steps,
                     parts);
  Group sym = gr, gen = gr;
  const int nsym = layout(&sym, [](const Mat& q) { return (q.mp / BT) * (q.mp / BT + 1) / 2; });
  const int ngen = layout(&gen, [](const Mat& q) { return (q.mp / BT) * (q.np / BT); });
  for (int t = 0; t < st.steps; ++t) {
    hipLaunchKernelGGL((product_kernel<T, BT, TO_S>), dim3(nsym), dim3(256), 0, s, sym, t, 0, 0.f, 0.f);
    hipLaunchKernelGGL((product_kernel<T, BT, TO_B>), dim3(nsym), dim3(256), 0, s, sym, t, 0, 0.f, 0.f);
    if (t + 1 < st.steps)
      hipLaunchKernelGGL((product_kernel<T, BT, TO_X>), dim3(ngen), dim3(256), 0, s, gen, t, t & 1, 0.f, 0.f);
    else
      hipLaunchKernelGGL((product_kernel<T, BT, MOM ? TO_PARAM : TO_OUT>), dim3(ngen), dim3(256), 0, s, gen, t, t & 1,
                         st.decay, st.rate);
  }
}

template <typename T, bool MOM>
int run_all(const void* const* src, void* const* dst, void* const* mom, const int* rows, const int* cols, int count,
            const Step& st, void* scratch, hipStream_t s) {
  for (int i0 = 0; i0 < count; i0 += GROUP) {
    Group gr;
    memset(&gr, 0, sizeof(gr));
    gr.count = count - i0 < GROUP ? count - i0 : GROUP;
    const int bt = tile_of(rows + i0, cols + i0, gr.count);
    char* at = static_cast<char*>(scratch);
    int parts = 0;
    for (int i = 0; i < gr.count; ++i) {
      Mat& q = gr.mat[i];
      shape_mat(&q, rows[i0 + i], cols[i0 + i], bt);
      q.g = src[i0 + i];
      q.out = dst[i0 + i];
      q.mom = mom ? static_cast<float*>(mom[i0 + i]) : nullptr;
      q.ws = at;
      at += mat_bytes(q);
      q.part0 = parts;
      parts += q.nparts;
      q.adjust = q.rows > q.cols ? sqrtf((float)q.rows / (float)q.cols) : 1.f;
    }
    launch_group<T, MOM, 64>(gr, st, reinterpret_cast<double*>(at), s);
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
  return scratch_bytes(rows_host, cols_host, count);
}

MMSA_EXPORT int mmsa_orthogonalize(const void* const* src_host, void* const* dst_host, const int* rows_host,
                                   const int* cols_host, int count, int dtype, int steps, float eps, void* scratch,
                                   void* stream) {
  if (int rc = check_sizes(rows_host, cols_host, count)) return rc;
  MMSA_REQUIRE(pointers_ok(src_host, count) && pointers_ok(dst_host, count) && scratch);
  MMSA_REQUIRE(((unsigned long long)scratch & 127) == 0 && steps >= 1 && steps <= MAX_STEPS && eps > 0.f);
  const Step st{0, 0.f, 1.f, 0, eps, 0.f, 0.f, steps};
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
  const Step st{1, (float)momentum, (float)(1.0 - momentum), nesterov, eps, (float)(1.0 - lr * weight_decay), (float)lr,
                steps};
  return run_all<float, true>(grads_host, params_host, momentum_host, rows_host, cols_host, count, st, scratch,
                              mmsa_stream(stream));
}
