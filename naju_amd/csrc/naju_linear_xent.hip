// naju_linear_xent.hip -- cross-entropy of a vocabulary head without its
// logits on MI355X (gfx950), behind the C ABI of include/naju_loss.h.
//
// With l = x W^T (x [n_rows, d], W [n_cols, d], 16 bits, products exact and
// sums in float32):
//   lse_m = log sum_v exp l[m][v],   loss_m = lse_m - l[m][target_m].
// Forward: each workgroup forms a tile of l in registers and leaves, for every
// row of it, the maximum and the sum of exponentials over the tile's columns;
// the lane that holds a row's target column writes that logit. A second kernel
// joins the tiles' pairs per row, a third forms the mean.
//
// Backward, with c_m the gradient of loss_m (0 for ignored rows):
//   dl[m][v] = c_m (exp(l[m][v] - lse_m) - [v = target_m])
//   dx = dl W,   dW = dl^T x.
// The vocabulary is taken in pieces. The forward's tile kernel forms a piece's
// logits again and writes dl for it in 16 bits; dW's rows of the piece are
// complete after one product over all rows; dx is summed over the pieces in
// float32. dl is rounded to 16 bits once, scaled so that the largest |c_m| is
// 2^14, which the products' epilogues take out again: c_m is 1 / n_rows under a
// mean, and a float16 dl would lose the small probabilities below its
// subnormals otherwise; and where all c_m are equal, as under a mean or a sum,
// a target's c_m (p - 1) near -c_m is then exact instead of off by the same
// rounding in every row (the gradients' error against float64 at 16384 x 768 x
// 50257 in bf16: 3.4e-3 with a power-of-two scale, 1.7e-3 so).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "gemm_few.h"
#include "gemm_out.h"
#include "naju_loss.h"
#include "naju_scan.h"

namespace naju_detail {
int loss_fail(int code, const char* fmt, ...);
void loss_clear();

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// (r, s) of a set of logits: r = max * log2 e, rounded, and the sum of
// 2^(v log2 e - r); the empty set is (-inf, 0). Every exponent is formed against
// that same r, so its rounding (2^-24 of a large maximum) is in the sum and in
// the target's exponent alike and out of their difference, the row's loss. A NaN
// among the values or an infinite maximum gives a NaN sum, as the softmax of
// such a row has.
__device__ __forceinline__ float ref_of(float r) { return r == -INFINITY ? 0.f : r; }
__device__ __forceinline__ void ms_join(float& r, float& s, float r2, float s2) {
  const float rn = fmaxf(r, r2), ref = ref_of(rn);
  s = s * __builtin_amdgcn_exp2f(r - ref) + s2 * __builtin_amdgcn_exp2f(r2 - ref);
  r = rn;
}

struct HeadArgs {
  const char* x;
  const char* w;       // the row of W behind the piece's first column
  int64_t x_ld, w_ld;  // bytes
  int64_t m, d, v;     // rows, contraction, columns of the piece
  int64_t v0;          // the piece's first column
  const int64_t* target;
  // forward
  float2* part;        // [tiles of n][m], of few rows [m][tiles]
  float* at_target;    // [m]
  // backward
  const float* lse;
  const float* coef;   // [m], scaled
  void* dl;            // [m][dl_ld], zero from v to dl_ld
  int64_t dl_ld;
};

template <typename T, typename C, bool BWD>
__global__ __launch_bounds__(C::kThreads, 2) void head_kernel(const HeadArgs g, int nm, int nn) {
  static_assert(C::TN == 4, "a wave's 64 columns are two groups of 32");
  NAJU_GEMM_LDS(C);
  __shared__ float2 s_ms[C::WN][C::BM];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wn = wave % C::WN, mt = (wave / C::WN) * C::TM * 16 + (lane & 15);
  const int steps = (int)((g.d + kBK - 1) / kBK);
  TilePipe<T, C, kAlongK, kAlongK> pipe;
  int bm = 0, bn = 0;
  const char *xb = nullptr, *wb = nullptr;
  auto a_at = [&](int s) { return Step{xb + (int64_t)s * (kBK * 2), g.d - (int64_t)s * kBK, 0}; };
  auto b_at = [&](int s) { return Step{wb + (int64_t)s * (kBK * 2), g.d - (int64_t)s * kBK, 0}; };
  auto begin = [&](int id) __attribute__((always_inline)) {
    tile_of(id, nm, nn, bm, bn);
    const int64_t m0 = (int64_t)bm * C::BM, n0 = (int64_t)bn * C::BN;
    const int ma = (int)(g.m - 1 - m0 < C::BM ? g.m - 1 - m0 : C::BM);
    const int na = (int)(g.v - 1 - n0 < C::BN ? g.v - 1 - n0 : C::BN);
    xb = g.x + m0 * g.x_ld;
    wb = g.w + n0 * g.w_ld;
    pipe.init((uint32_t)g.x_ld, (uint32_t)g.w_ld, [&](int r) { return r < ma ? r : ma; },
              [&](int r) {
                const int n = wide_row(r);
                return n < na ? n : na;
              });
    pipe.start(s_steps, steps, a_at, b_at);
  };
  int id = blockIdx.x;
  begin(id);
  for (;;) {
    acc_t acc[C::TM][C::TN];
    pipe.run(acc, s_steps, steps, a_at, b_at);
    const int64_t m0 = (int64_t)bm * C::BM, n0 = (int64_t)bn * C::BN;
    const int tile_n = bn;
    id += gridDim.x;
    const bool more = id < nm * nn;
    if (more) begin(id);
    // acc[i][j][r] is column nw + col(j, r)
    const int64_t nw = n0 + wn * 64 + 8 * (lane >> 4);
    auto col = [](int j, int r) { return (j >> 1) * 32 + (j & 1) * 4 + r; };
    if constexpr (!BWD) {
      // columns past the end take no part
      if (n0 + C::BN > g.v) {
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (nw + col(j, r) >= g.v) {
#pragma unroll
              for (int i = 0; i < C::TM; ++i) acc[i][j][r] = -INFINITY;
            }
      }
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int64_t m = m0 + mt + i * 16;
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float top = mx * kLog2e, ref = ref_of(top);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], kLog2e, -ref));
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (lane < 16) s_ms[wn][mt + i * 16] = make_float2(top, s);
        if (m < g.m) {
          const int64_t target = g.target[m], t = target - nw;
          if (t >= 0 && t < 64 && target < g.v) {
            // the lane that holds the target's column (if this one does)
#pragma unroll
            for (int j = 0; j < C::TN; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (t == col(j, r)) g.at_target[m] = acc[i][j][r];
          }
        }
      }
      __syncthreads();
      for (int r = threadIdx.x; r < C::BM; r += C::kThreads) {
        if (m0 + r >= g.m) break;
        float2 a = s_ms[0][r];
#pragma unroll
        for (int w = 1; w < C::WN; ++w) {
          const float2 b = s_ms[w][r];
          ms_join(a.x, a.y, b.x, b.y);
        }
        g.part[(int64_t)tile_n * g.m + m0 + r] = a;
      }
      // the next tile's s_ms is written behind its run()'s barriers
    } else {
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int64_t m = m0 + mt + i * 16;
        if (m >= g.m) continue;
        const float c = g.coef[m], lse = g.lse[m];
        const int64_t t = g.target[m] - g.v0 - nw;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t n = nw + h * 32;
          if (n >= g.dl_ld) continue;
          float o[8];
          // (the difference first: it is exact near lse, and p of a row's one class 1)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            o[e] = __builtin_amdgcn_exp2f((acc[i][2 * h + (e >> 2)][e & 3] - lse) * kLog2e);
          // few waves hold a target here, and only the last tiles columns past the end
          const int64_t th = t - h * 32;
          if (__ballot(th >= 0 && th < 8)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] -= th == e ? 1.f : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] *= c;
          if (n0 + C::BN > g.v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = n + e < g.v ? o[e] : 0.f;
          }
          // an ignored row's gradient is 0 whatever its logits are
          typedef typename UserVec<T, 8, sizeof(T)>::type vec;
          typedef uint32_t u4 __attribute__((ext_vector_type(4)));
          vec v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (T)o[e];
          const u4 bits = __builtin_bit_cast(u4, v);
          *reinterpret_cast<vec*>((T*)g.dl + m * g.dl_ld + n) =
              __builtin_bit_cast(vec, c != 0.f ? bits : u4{0, 0, 0, 0});
        }
      }
    }
    if (!more) break;
  }
}

// Forward for at most 16 MT rows: kFewCols columns a workgroup, eight waves (16
// rows, d = 768, with the join, over 4096 / 50257 classes 8.3 / 25.2 us; 64 columns by
// four waves 10.9 / 28.0, 16 by eight 9.1 / 30.5).
constexpr int kFewCols = 32, kFewThreads = 512;
template <typename T, int MT>
__global__ __launch_bounds__(kFewThreads) void head_few_kernel(const HeadArgs g) {
  typedef FewProduct<T, kFewCols / 16, MT, kFewThreads / 64> P;
  __shared__ float s[P::kFloats];
  const int64_t n0 = (int64_t)blockIdx.x * P::N;
  P::run(
      s, g.d, [&](int r) { return g.x + (r < g.m ? r : g.m - 1) * g.x_ld; },
      [&](int r) { return g.w + (n0 + r < g.v ? n0 + r : g.v - 1) * g.w_ld; });
  // kSlices neighbouring lanes share a row
  constexpr int kSlices = P::kThreads / P::M;
  static_assert(kSlices >= 4 && kSlices <= 64, "a row's lanes lie in one wave");
  const int m = threadIdx.x / kSlices, q = threadIdx.x % kSlices;
  const int64_t target = m < g.m ? g.target[m] : -1;
  float r = -INFINITY, sum = 0.f;
  for (int n = q; n < P::N; n += kSlices)
    if (n0 + n < g.v) {
      const float v = s[n * P::M + m];
      if (n0 + n == target) g.at_target[m] = v;
      // (fmaxf leaves a NaN out of r; it reaches the sum)
      const float rn = fmaxf(r, fmaxf(v, -INFINITY) * kLog2e), ref = ref_of(rn);
      sum = sum * __builtin_amdgcn_exp2f(r - ref) + __builtin_amdgcn_exp2f(fmaf(v, kLog2e, -ref));
      r = rn;
    }
#pragma unroll
  for (int h = kSlices / 2; h >= 1; h >>= 1) {
    const float r2 = __shfl_xor(r, h, 64), sum2 = __shfl_xor(sum, h, 64);
    ms_join(r, sum, r2, sum2);
  }
  if (q == 0 && m < g.m) g.part[(int64_t)m * gridDim.x + blockIdx.x] = make_float2(r, sum);
}

// Joins the tiles' pairs of a row: R rows a workgroup, 1024 / R lanes of it a
// row, each taking every (1024 / R)th tile (four loaded before the first is
// joined). One row at a time (few rows): the pairs of a row lie together.
template <int R>
__global__ __launch_bounds__(1024) void head_join_kernel(const float2* __restrict__ part, int tiles,
                                                         const float* __restrict__ at_target,
                                                         const int64_t* __restrict__ target, int64_t rows, int64_t cols,
                                                         int64_t ignore, float* __restrict__ lse,
                                                         float* __restrict__ row_loss) {
  constexpr int kLanes = 1024 / R;
  static_assert(R == 1 || R == 16, "one row, or one for each wave");
  __shared__ float2 s_ms[R == 1 ? 16 : 64][R + 1];
  const int row = threadIdx.x % R, q = threadIdx.x / R;
  const int64_t m = (int64_t)blockIdx.x * R + row;
  const int64_t mc = m < rows ? m : rows - 1;
  float r = -INFINITY, s = 0.f;
  for (int t0 = q; t0 < tiles; t0 += 4 * kLanes) {
    float2 p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + u * kLanes;
      const int tc = t < tiles ? t : t0;
      p[u] = part[R == 1 ? mc * tiles + tc : tc * rows + mc];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (t0 + u * kLanes < tiles) ms_join(r, s, p[u].x, p[u].y);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto join_lanes = [&](int n) {
#pragma unroll
    for (int h = n / 2; h >= 1; h >>= 1) {
      const float r2 = __shfl_xor(r, h, 64), s2 = __shfl_xor(s, h, 64);
      ms_join(r, s, r2, s2);
    }
  };
  if constexpr (R == 1) {
    // the waves' pairs, then the first wave's lanes join those
    join_lanes(64);
    if (lane == 0) s_ms[wave][0] = make_float2(r, s);
    __syncthreads();
    const float2 p = s_ms[lane & 15][0];
    r = p.x;
    s = p.y;
    join_lanes(16);
  } else {
    // wave w joins the 64 pairs of row w
    s_ms[q][row] = make_float2(r, s);
    __syncthreads();
    const float2 p = s_ms[lane][wave];
    r = p.x;
    s = p.y;
    join_lanes(64);
  }
  const int64_t mw = (int64_t)blockIdx.x * R + (R == 1 ? 0 : wave);
  if ((R == 1 ? threadIdx.x : lane) != 0 || mw >= rows) return;
  const float ref = ref_of(r);
  const double log2s = (double)__builtin_amdgcn_logf(s), scale = 1.0 / (double)kLog2e;
  lse[mw] = (float)(((double)ref + log2s) * scale);
  const int64_t t = target[mw];
  // ignored rows are 0; a target outside the vocabulary is NaN
  row_loss[mw] = t == ignore ? 0.f
                 : t >= 0 && t < cols ? (float)((log2s - (double)fmaf(at_target[mw], kLog2e, -ref)) * scale)
                                      : __builtin_nanf("");
}

// loss = the rows' sum (in float64, in a fixed order) times scale, with
// scale = 1 / #valid rows (mean) or 1. No valid row gives a NaN mean.
__global__ __launch_bounds__(1024) void head_sum_kernel(const float* __restrict__ row_loss,
                                                        const int64_t* __restrict__ target, int64_t rows,
                                                        int64_t ignore, int mean, float* __restrict__ loss,
                                                        float* __restrict__ scale) {
  __shared__ double s_sum[1024];
  __shared__ int64_t s_n[1024];
  double sum = 0.0;
  int64_t n = 0;
  for (int64_t m = threadIdx.x; m < rows; m += 1024) {
    sum += (double)row_loss[m];
    n += target[m] != ignore;
  }
  s_sum[threadIdx.x] = sum;
  s_n[threadIdx.x] = n;
  for (int h = 512; h > 0; h >>= 1) {
    __syncthreads();
    if (threadIdx.x < h) {
      s_sum[threadIdx.x] += s_sum[threadIdx.x + h];
      s_n[threadIdx.x] += s_n[threadIdx.x + h];
    }
  }
  if (threadIdx.x == 0) {
    loss[0] = mean ? (float)(s_sum[0] / (double)s_n[0]) : (float)s_sum[0];
    scale[0] = mean ? (float)(1.0 / (double)s_n[0]) : 1.f;
  }
}

// What the backward's products take of the rows' gradients c_m = scale dloss:
// coef[m] = 2^14 c_m / max |c| for valid rows, 0 for ignored ones, NaN for a
// target outside the vocabulary; unscale = max |c| / 2^14. Zero, infinite and
// near-subnormal gradients stay as they are.
__device__ __forceinline__ float coef_top(float mx) { return mx > 1e-30f && mx < 1e30f ? mx : 16384.f; }
__device__ __forceinline__ float coef_of(float c, float top, int64_t t, int64_t cols, int64_t ignore) {
  return t == ignore ? 0.f : (t >= 0 && t < cols ? c / top * 16384.f : __builtin_nanf(""));
}

// For a gradient of its own for every row: the largest first.
__global__ __launch_bounds__(1024) void head_coef_kernel(const float* __restrict__ dloss,
                                                         const float* __restrict__ scale,
                                                         const int64_t* __restrict__ target, int64_t rows,
                                                         int64_t cols, int64_t ignore, float* __restrict__ coef,
                                                         float* __restrict__ unscale) {
  __shared__ float s_max[16];
  const float sc = scale ? scale[0] : 1.f;
  float mx = 0.f;
  for (int64_t m = threadIdx.x; m < rows; m += 1024)
    if (target[m] != ignore) mx = fmaxf(mx, fabsf(dloss[m] * sc));
#pragma unroll
  for (int h = 32; h >= 1; h >>= 1) mx = fmaxf(mx, __shfl_xor(mx, h, 64));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) mx = fmaxf(mx, s_max[w]);
  const float top = coef_top(mx);
  for (int64_t m = threadIdx.x; m < rows; m += 1024)
    coef[m] = coef_of(dloss[m] * sc, top, target[m], cols, ignore);
  if (threadIdx.x == 0) unscale[0] = top * (1.f / 16384.f);
}

// xm = x with the rows of ignored targets zero, rows of round_up(d, 8): what
// an ignored row holds (padding may hold anything, NaN included) stays out of
// dW's sum over rows, where 0 * NaN would not. With one gradient for all rows
// (dloss not null) coef and unscale are formed here too.
__global__ __launch_bounds__(256) void head_mask_kernel(const uint16_t* __restrict__ x, int64_t x_ld,
                                                        const int64_t* __restrict__ target, int64_t rows, int64_t d8,
                                                        int64_t cols, int64_t ignore, uint16_t* __restrict__ xm,
                                                        const float* __restrict__ dloss,
                                                        const float* __restrict__ scale, float* __restrict__ coef,
                                                        float* __restrict__ unscale) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const int64_t per = d8 / 8, n = rows * per, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t hop = (int64_t)gridDim.x * 256;
  for (int64_t i = first; i < n; i += hop) {
    const int64_t r = i / per, c = (i - r * per) * 8;
    const u4 v = *reinterpret_cast<const u4*>(x + r * x_ld + c);
    *reinterpret_cast<u4*>(xm + i * 8) = target[r] == ignore ? u4{0, 0, 0, 0} : v;
  }
  if (!dloss) return;
  const float c = dloss[0] * (scale ? scale[0] : 1.f), top = coef_top(fabsf(c));
  for (int64_t m = first; m < rows; m += hop) coef[m] = coef_of(c, top, target[m], cols, ignore);
  if (first == 0) unscale[0] = top * (1.f / 16384.f);
}

// ------------------------------------------------------------------ host side

// The large tile where the small ones, two a CU, would need a second round. Both
// measured over 48 to 512 large tiles, 240 to 16368 rows, d = 256, 768 and 2048
// (1008 rows, d = 768; large and small): forward 96 tiles 24.5 and 20.0 us, 128 27.1
// and 24.7, 144 28.0 and 33.8, 256 31.3 and 42.8, 512 56.2 and 74.8; gradient of the
// logits 128 29.5 and 26.0, 144 29.5 and 33.0, 256 35.1 and 51.6, 512 63.1 and 98.4.
// The rule loses where the large tiles have just begun a second round themselves,
// 257 to about 300 of them: at d = 768 up to 11% (288 tiles of 4080 rows forward 46.3
// and 42.2), at d = 2048 up to 5%, at d = 256 up to 17% forward and 21% for the
// gradient, and 10% there from 301 to 512 tiles.
bool head_large(int64_t m, int64_t v) { return ceil_div(m, TileL::BM) * ceil_div(v, TileL::BN) > kCUs / 2; }

// Few rows: bound by the loads of W. With the join, here and on the tiles below,
// cold weights, d = 768 / 2048 / 4096: 1 row over 4096 classes 7.0 / 10.7 / 15.9 and
// 12.6 / 31.6 / 56.6 us, over 50257 19.9 / 45.0 / 89.9 and 29.2 / 61.2 / 106; 16 rows
// 8.1 / 13.0 / 19.7 and 12.9 / 32.0 / 56.9, 25.2 / 57.8 / 109 and 29.5 / 61.5 / 110, over
// 131072 51.6 / 127 / 247 and 59.5 / 139 / 238 (the only loss to 16 rows, 4%); 32 rows
// over 24576 17.3 / 35.8 / 64.1 and 18.8 / 36.3 / 63.3, 50257 29.8 / 68.5 / 132 and 30.1 /
// 62.0 / 110; 64 rows over 4096 11.2 / 19.4 / 32.0 and 13.8 / 32.9 / 57.8, 12347 19.1 / 33.8
// / 59.0 and 18.2 / 34.3 / 60.9. (A launch has fewer than 2^32 threads, 16 a column here.)
bool head_few(int64_t m, int64_t v) {
  return (m <= 16 && v <= 1 << 27) || (m <= 32 && v <= 24576) || (m <= 64 && v <= 8192);
}

template <typename T, bool BWD>
void head_launch(const HeadArgs& g, hipStream_t st) {
  if (!BWD && head_few(g.m, g.v)) {
    const unsigned grid = (unsigned)ceil_div(g.v, kFewCols);
    if (g.m <= 16)
      head_few_kernel<T, 1><<<grid, kFewThreads, 0, st>>>(g);
    else if (g.m <= 32)
      head_few_kernel<T, 2><<<grid, kFewThreads, 0, st>>>(g);
    else
      head_few_kernel<T, 4><<<grid, kFewThreads, 0, st>>>(g);
    return;
  }
  // backward tiles also cover the zero columns up to dl_ld
  const int64_t v = BWD ? g.dl_ld : g.v;
  if (head_large(g.m, v)) {
    const int nm = (int)ceil_div(g.m, TileL::BM), nn = (int)ceil_div(v, TileL::BN);
    head_kernel<T, TileL, BWD><<<tile_grid<TileL>(nm * nn), TileL::kThreads, 0, st>>>(g, nm, nn);
  } else {
    const int nm = (int)ceil_div(g.m, TileS::BM), nn = (int)ceil_div(v, TileS::BN);
    head_kernel<T, TileS, BWD><<<tile_grid<TileS>(nm * nn), TileS::kThreads, 0, st>>>(g, nm, nn);
  }
}

int launched() {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return loss_fail(NAJU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
  return NAJU_OK;
}

int check_head(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const int64_t* target, int64_t n_rows,
               int64_t d, int64_t n_cols, int dtype) {
  if (n_rows < 0 || d < 1 || n_cols < 1)
    return loss_fail(NAJU_ERR_INVALID, "n_rows must be >= 0, d and n_cols positive");
  if (dtype != NAJU_DTYPE_BF16 && dtype != NAJU_DTYPE_F16)
    return loss_fail(NAJU_ERR_UNSUPPORTED, "the head's loss serves bf16 and f16");
  // (a launch has fewer than 2^32 threads: 64 a row in the join)
  if (n_rows > (1 << 25) || d > (1 << 21) || n_cols > (1 << 29) || x_ld > (1 << 21) || w_ld > (1 << 21) ||
      !tiles_fit(n_rows, n_cols))
    return loss_fail(NAJU_ERR_UNSUPPORTED,
                     "shape too large (n_rows up to 2^25, n_cols to 2^29, d and row strides to 2^21 elements)");
  const int64_t d8 = round_up(d, 8);
  if (x_ld < d8 || w_ld < d8 || x_ld % 8 || w_ld % 8)
    return loss_fail(NAJU_ERR_INVALID, "row strides must be multiples of 8, at least d rounded up to 8");
  if (n_rows == 0) return NAJU_OK;
  if (!x || !w || !target) return loss_fail(NAJU_ERR_INVALID, "null pointer (x, w and target are required)");
  if (((uintptr_t)x | (uintptr_t)w) & 15) return loss_fail(NAJU_ERR_INVALID, "x and w must be 16-byte aligned");
  return NAJU_OK;
}

int64_t head_tiles(int64_t m, int64_t v) {
  if (head_few(m, v)) return ceil_div(v, kFewCols);
  return ceil_div(v, head_large(m, v) ? TileL::BN : TileS::BN);
}

size_t head_fwd_bytes(int64_t m, int64_t v) {
  return (size_t)(round_up(head_tiles(m, v) * m * 8, 256) + round_up(m * 4, 256));
}

// Bytes of dl that one piece of the vocabulary may take (of 288 GB).
constexpr int64_t kPieceBytes = 1ll << 30;

struct HeadBwdPlan {
  int64_t piece;  // columns of a piece, a multiple of 256
  int pieces;
  GemmPlan dx, dw;
  size_t o_xm, o_coef, o_acc, o_part, total;
};
HeadBwdPlan head_bwd_plan(int64_t m, int64_t d, int64_t v) {
  HeadBwdPlan p;
  int64_t most = kPieceBytes / (2 * (m > 0 ? m : 1)) / 256 * 256;
  if (most < 256) most = 256;
  // in several pieces, each (but the last) a whole number of rounds of 256 x 256
  // tiles of dW over the CUs, where the bytes allow one
  const int64_t round = kCUs / ceil_div(d, 256) * 256;
  p.piece = v <= most ? round_up(v, 256) : (round > 0 && most >= round ? most / round * round : most);
  p.pieces = (int)ceil_div(v, p.piece);
  p.dx = gemm_plan(m, d, p.piece < v ? p.piece : v, 0);
  p.dw = gemm_plan(p.piece < v ? p.piece : v, d, m, 0);
  p.o_xm = (size_t)round_up(m * p.piece * 2, 256);
  p.o_coef = p.o_xm + (size_t)round_up(m * round_up(d, 8) * 2, 256);
  p.o_acc = p.o_coef + (size_t)round_up(m * 4, 256) + 256;
  p.o_part = p.o_acc + (p.pieces > 1 ? (size_t)round_up(m * d * 4, 256) : 0);
  const size_t a = gemm_part_bytes(p.dx, m, d), b = gemm_part_bytes(p.dw, p.piece, d);
  p.total = p.o_part + (a > b ? a : b) + 256;
  return p;
}

template <typename T, typename TW>
int head_bwd(HeadArgs g, const HeadBwdPlan& p, int64_t v, void* dx, void* dw, char* ws, hipStream_t st) {
  const char* w = g.w;
  const float* unscale = (const float*)(ws + p.o_acc - 256);
  for (int i = 0; i < p.pieces; ++i) {
    g.v0 = i * p.piece;
    g.v = v - g.v0 < p.piece ? v - g.v0 : p.piece;
    g.w = w + g.v0 * g.w_ld;
    g.dl_ld = round_up(g.v, 64);
    head_launch<T, true>(g, st);
    if (int rc = launched()) return rc;
    if (dx) {
      GemmOut o = {};
      o.a = (const char*)g.dl;
      o.lda = g.dl_ld * 2;
      o.b[0] = o.b[1] = g.w;
      o.ldb = g.w_ld;
      o.k_first = g.v;
      o.m = g.m;
      o.n = g.d;
      o.part = (float*)(ws + p.o_part);
      o.out[0] = dx;
      o.ldo = g.d;
      o.m_half = o.out_rows = g.m;
      o.scale = unscale;
      o.acc = (float*)(ws + p.o_acc);
      o.acc_in = i > 0;
      o.acc_out = i + 1 < p.pieces;
      // the last piece may be shorter: a plan of its own, with no more splits
      GemmPlan q = gemm_plan(g.m, g.d, g.v, 0);
      if (q.splits > p.dx.splits) q = p.dx;
      gemm_out_launch<T, T, kAlongK>(o, q, st);
      if (int rc = launched()) return rc;
    }
    if (dw) {
      GemmOut o = {};
      o.a = (const char*)g.dl;
      o.lda = g.dl_ld * 2;
      o.b[0] = o.b[1] = g.x;
      o.ldb = g.x_ld;
      o.k_first = g.m;
      o.m = g.v;
      o.n = g.d;
      o.part = (float*)(ws + p.o_part);
      o.out[0] = (TW*)dw + g.v0 * g.d;
      o.ldo = g.d;
      o.m_half = o.out_rows = g.v;
      o.scale = unscale;
      GemmPlan q = gemm_plan(g.v, g.d, g.m, 0);
      if (gemm_part_bytes(q, g.v, g.d) > p.total - 256 - p.o_part) q = p.dw;
      gemm_out_launch<T, TW, kAlongMN>(o, q, st);
      if (int rc = launched()) return rc;
    }
  }
  return NAJU_OK;
}

}  // namespace
}  // namespace naju_detail

using namespace naju_detail;

extern "C" {

size_t naju_linear_xent_workspace_bytes(int64_t n_rows, int64_t d, int64_t n_cols, int backward) {
  if (n_rows < 0 || d < 1 || n_cols < 1) return 0;
  return backward ? head_bwd_plan(n_rows, d, n_cols).total : head_fwd_bytes(n_rows, n_cols) + 256;
}

int naju_linear_xent_fwd(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const int64_t* target,
                         int64_t n_rows, int64_t d, int64_t n_cols, int dtype, int64_t ignore_index, float* lse,
                         float* row_loss, int mean, float* loss, float* scale, void* workspace, size_t workspace_bytes,
                         void* stream) {
  loss_clear();
  int rc = check_head(x, x_ld, w, w_ld, target, n_rows, d, n_cols, dtype);
  if (rc) return rc;
  if (!loss != !scale) return loss_fail(NAJU_ERR_INVALID, "loss and scale come together");
  if (n_rows > 0 && (!lse || !row_loss)) return loss_fail(NAJU_ERR_INVALID, "null pointer (lse and row_loss)");
  hipStream_t st = (hipStream_t)stream;
  if (n_rows > 0) {
    const size_t need = head_fwd_bytes(n_rows, n_cols);
    if (!workspace || workspace_bytes < need) return loss_fail(NAJU_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
    if ((uintptr_t)workspace & 255) return loss_fail(NAJU_ERR_INVALID, "workspace must be 256-byte aligned");
    const int64_t tiles = head_tiles(n_rows, n_cols);
    HeadArgs g = {};
    g.x = (const char*)x;
    g.w = (const char*)w;
    g.x_ld = x_ld * 2;
    g.w_ld = w_ld * 2;
    g.m = n_rows;
    g.d = d;
    g.v = n_cols;
    g.target = target;
    g.part = (float2*)workspace;
    g.at_target = (float*)((char*)workspace + round_up(tiles * n_rows * 8, 256));
    if (dtype == NAJU_DTYPE_BF16)
      head_launch<bf16_t, false>(g, st);
    else
      head_launch<f16_t, false>(g, st);
    if ((rc = launched())) return rc;
    // 16 rows a workgroup read whole lines of the pairs; the many tiles of few rows
    // want all its lanes on one (16 rows of 786 tiles 5.0 us, one by one with 1571 3.9)
    if (head_few(n_rows, n_cols))
      head_join_kernel<1><<<(unsigned)n_rows, 1024, 0, st>>>(g.part, (int)tiles, g.at_target, target, n_rows, n_cols,
                                                             ignore_index, lse, row_loss);
    else
      head_join_kernel<16><<<(unsigned)ceil_div(n_rows, 16), 1024, 0, st>>>(g.part, (int)tiles, g.at_target, target, n_rows,
                                                                            n_cols, ignore_index, lse, row_loss);
    if ((rc = launched())) return rc;
  }
  if (loss) {
    head_sum_kernel<<<1, 1024, 0, st>>>(row_loss, target, n_rows, ignore_index, mean, loss, scale);
    return launched();
  }
  return NAJU_OK;
}

int naju_linear_xent_bwd(const void* x, int64_t x_ld, const void* w, int64_t w_ld, const int64_t* target,
                         int64_t n_rows, int64_t d, int64_t n_cols, int dtype, int64_t ignore_index, const float* lse,
                         const float* scale, const float* dloss, int64_t dloss_step, void* dx, void* dw, int dw_dtype,
                         void* workspace, size_t workspace_bytes, void* stream) {
  loss_clear();
  int rc = check_head(x, x_ld, w, w_ld, target, n_rows, d, n_cols, dtype);
  if (rc) return rc;
  if (dw_dtype != dtype && dw_dtype != NAJU_DTYPE_F32)
    return loss_fail(NAJU_ERR_INVALID, "dw_dtype must be the operands' dtype or f32");
  if (dloss_step != 0 && dloss_step != 1) return loss_fail(NAJU_ERR_INVALID, "dloss_step must be 0 or 1");
  if (n_rows == 0) return NAJU_OK;
  if (!lse || !dloss) return loss_fail(NAJU_ERR_INVALID, "null pointer (lse and dloss are required)");
  const HeadBwdPlan p = head_bwd_plan(n_rows, d, n_cols);
  if (!workspace || workspace_bytes < p.total)
    return loss_fail(NAJU_ERR_WORKSPACE, "workspace of %zu bytes needed", p.total);
  if ((uintptr_t)workspace & 255) return loss_fail(NAJU_ERR_INVALID, "workspace must be 256-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  float *coef = (float*)(ws + p.o_coef), *unscale = (float*)(ws + p.o_acc - 256);
  if (dloss_step) {
    head_coef_kernel<<<1, 1024, 0, st>>>(dloss, scale, target, n_rows, n_cols, ignore_index, coef, unscale);
    if ((rc = launched())) return rc;
  }
  const int64_t d8 = round_up(d, 8), wgs = ceil_div(n_rows * (d8 / 8), 256);
  head_mask_kernel<<<dim3((unsigned)(wgs < 2048 ? wgs : 2048)), 256, 0, st>>>(
      (const uint16_t*)x, x_ld, target, n_rows, d8, n_cols, ignore_index, (uint16_t*)(ws + p.o_xm),
      dloss_step ? nullptr : dloss, scale, coef, unscale);
  if ((rc = launched())) return rc;
  HeadArgs g = {};
  g.x = ws + p.o_xm;
  g.w = (const char*)w;
  g.x_ld = d8 * 2;
  g.w_ld = w_ld * 2;
  g.m = n_rows;
  g.d = d;
  g.target = target;
  g.lse = lse;
  g.coef = coef;
  g.dl = ws;
  if (dtype == NAJU_DTYPE_BF16)
    return dw_dtype == NAJU_DTYPE_F32 ? head_bwd<bf16_t, float>(g, p, n_cols, dx, dw, ws, st)
                                      : head_bwd<bf16_t, bf16_t>(g, p, n_cols, dx, dw, ws, st);
  return dw_dtype == NAJU_DTYPE_F32 ? head_bwd<f16_t, float>(g, p, n_cols, dx, dw, ws, st)
                                    : head_bwd<f16_t, f16_t>(g, p, n_cols, dx, dw, ws, st);
}

}  // extern "C"
