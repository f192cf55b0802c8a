// naju_norm.hip -- layer norm and its gradients on MI355X (gfx950), and the
// padded row copy of the 16-bit products, behind the C ABI of
// include/naju_mixer.h.
//
//   y = (x - mean) rstd * w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
// and, with xh = (x - mean) rstd and g = dy * w,
//   dx = rstd (g - mean(g) - xh mean(g xh)) [+ dres],
//   dw = sum_rows dy xh,   db = sum_rows dy.
//
// Bound by memory both ways: x is read once and y written once forward; x, dy
// (and dres) are read once and dx written once backward. A row is held in the
// registers of one wave (up to 2048 columns forward, 1024 backward) or of the
// four waves of a workgroup (up to 16384), eight neighbouring values a lane, so the mean and
// then the centred square sum are exact two-pass statistics in float32 at one
// read; wider rows are read again for each. The backward keeps its dw and db
// terms in registers over all the rows of a wave and leaves one row of sums a
// workgroup, which a second kernel adds in order: deterministic.
//
// Rows may start at any element: vectors are loaded with their element's
// alignment.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "naju_mixer.h"
#include "naju_scan.h"
#include "scan_internal.h"

namespace naju_detail {
int mixer_fail(int code, const char* fmt, ...);
void mixer_clear();

namespace {

constexpr int kV = 8;  // values of a row a lane holds together

// Eight neighbouring values from column c of a row of d (0 past the end).
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t d, float (&v)[kV]) {
  typedef typename UserVec<T, kV, sizeof(T)>::type v8;
  if (c + kV <= d) {
    const v8 o = *reinterpret_cast<const v8*>(row + c);
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = (float)o[e];
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e) v[e] = c + e < d ? (float)row[c + e] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int64_t c, int64_t d, const float (&v)[kV]) {
  typedef typename UserVec<T, kV, sizeof(T)>::type v8;
  if (c + kV <= d) {
    v8 o;
#pragma unroll
    for (int e = 0; e < kV; ++e) o[e] = (T)v[e];
    *reinterpret_cast<v8*>(row + c) = o;
  } else {
#pragma unroll
    for (int e = 0; e < kV; ++e)
      if (c + e < d) row[c + e] = (T)v[e];
  }
}

// The sums over the WPR waves that hold a row, in every lane: one barrier, with
// two sets of slots that calls use in turn.
template <int WPR>
__device__ __forceinline__ float2 row_sums(float a, float b, float2 (&s_red)[2][4], int turn) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    a += __shfl_xor(a, m, 64);
    b += __shfl_xor(b, m, 64);
  }
  if constexpr (WPR == 1) return make_float2(a, b);
  float2(&red)[4] = s_red[turn & 1];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(a, b);
  __syncthreads();
  return make_float2(red[0].x + red[1].x + red[2].x + red[3].x, red[0].y + red[1].y + red[2].y + red[3].y);
}
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float2 (&s_red)[2][4], int turn) {
  return row_sums<WPR>(v, 0.f, s_red, turn).x;
}

// The columns of a lane's group k: kV from `base` on, of which those before
// `first` belong to the lane before it. Groups past the row's end start at its
// last kV columns (d >= kV) and own none; the group that reaches past it starts
// there too and owns what is left. So every load and store is one whole
// vector, and what two lanes store twice is the same value.
template <int WPR>
struct Cols {
  int64_t base;
  int first;
  __device__ __forceinline__ Cols(int k, int t, int64_t d) {
    const int64_t c = (int64_t)(k * 64 * WPR + t) * kV;
    base = c < d - kV ? c : d - kV;
    first = c - base < kV ? (int)(c - base) : kV;
  }
  __device__ __forceinline__ bool owns(int e) const { return e >= first; }
  __device__ __forceinline__ bool any() const { return first < kV; }
};
template <typename T>
struct Vec8 {
  typedef typename UserVec<T, kV, sizeof(T)>::type type;
  static __device__ __forceinline__ type load(const T* p) { return *reinterpret_cast<const type*>(p); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[kV]) {
    type o;
#pragma unroll
    for (int e = 0; e < kV; ++e) o[e] = (T)v[e];
    *reinterpret_cast<type*>(p) = o;
  }
};

struct NormArgs {
  const void* x;
  const float* w;  // or null: 1
  const float* b;  // or null: 0
  int64_t x_ld, rows, d;
  float eps;
  void* y;
  float* mean;
  float* rstd;
  const void* dy;
  int64_t dy_ld;
  const void* dres;  // or null
  void* dx;
  float* part;  // [grid][2][d], or null
};

constexpr int kWaves = 4;  // waves of a workgroup

// WPR: waves per row (1 or kWaves); G: groups of kV values a lane.
template <typename TX, typename TY, int WPR, int G>
__global__ __launch_bounds__(64 * kWaves) void norm_fwd_kernel(const NormArgs g) {
  __shared__ float2 s_red[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = WPR == 1 ? (int64_t)blockIdx.x * kWaves + wave : blockIdx.x;
  if (r >= g.rows) return;  // with WPR == kWaves: never
  const int t = WPR == 1 ? lane : (int)threadIdx.x;
  const TX* row = (const TX*)g.x + r * g.x_ld;
  typename Vec8<TX>::type raw[G];
#pragma unroll
  for (int k = 0; k < G; ++k) raw[k] = Vec8<TX>::load(row + Cols<WPR>(k, t, g.d).base);
  float v[G][kV];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const Cols<WPR> c(k, t, g.d);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      v[k][e] = (float)raw[k][e];
      s += c.owns(e) ? v[k][e] : 0.f;
    }
  }
  const float mean = row_sum<WPR>(s, s_red, 0) / (float)g.d;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const Cols<WPR> c(k, t, g.d);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      v[k][e] -= mean;
      s = fmaf(c.owns(e) ? v[k][e] : 0.f, v[k][e], s);
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<WPR>(s, s_red, 1) / (float)g.d + g.eps);
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const Cols<WPR> c(k, t, g.d);
    if (!c.any()) continue;
    typename Vec8<float>::type w, b;
    if (g.w) w = Vec8<float>::load(g.w + c.base);
    if (g.b) b = Vec8<float>::load(g.b + c.base);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      float o = v[k][e] * rstd;
      if (g.w) o *= w[e];
      if (g.b) o += b[e];
      v[k][e] = o;
    }
    Vec8<TY>::store((TY*)g.y + r * g.d + c.base, v[k]);
  }
  if (t == 0 && g.mean) {
    g.mean[r] = mean;
    g.rstd[r] = rstd;
  }
}

// Each row group (a wave, or the workgroup) takes rows gridDim.x * (row groups
// a workgroup) apart, the next row's values loaded before this one's are used.
template <typename TX, typename TY, int WPR, int G>
__global__ __launch_bounds__(64 * kWaves) void norm_bwd_kernel(const NormArgs g) {
  __shared__ float2 s_red[2][4];
  __shared__ float s_acc[WPR == 1 ? kWaves : 1][WPR == 1 ? G * 64 * kV : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = WPR == 1 ? lane : (int)threadIdx.x;
  const int64_t first = WPR == 1 ? (int64_t)blockIdx.x * kWaves + wave : blockIdx.x;
  const int64_t stride = (int64_t)gridDim.x * (WPR == 1 ? kWaves : 1);
  const float inv_d = 1.f / (float)g.d;
  float aw[G][kV], ab[G][kV];
  typename Vec8<TX>::type nx[G];
  typename Vec8<TY>::type ny[G];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t r) {
    nmean = g.mean[r];
    nrstd = g.rstd[r];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const int64_t c = Cols<WPR>(k, t, g.d).base;
      nx[k] = Vec8<TX>::load((const TX*)g.x + r * g.x_ld + c);
      ny[k] = Vec8<TY>::load((const TY*)g.dy + r * g.dy_ld + c);
    }
  };
#pragma unroll
  for (int k = 0; k < G; ++k)
#pragma unroll
    for (int e = 0; e < kV; ++e) aw[k][e] = ab[k][e] = 0.f;
  int turn = 0;
  if (first < g.rows) fetch(first);
  for (int64_t r = first; r < g.rows; r += stride) {
    float xh[G][kV], dy[G][kV];
    const float mean = nmean, rstd = nrstd;
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        xh[k][e] = ((float)nx[k][e] - mean) * rstd;
        dy[k][e] = (float)ny[k][e];
      }
    fetch(r + stride < g.rows ? r + stride : r);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const Cols<WPR> c(k, t, g.d);
      typename Vec8<float>::type w;
      if (g.w) w = Vec8<float>::load(g.w + c.base);
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        // (only owned columns' sums are kept)
        ab[k][e] += dy[k][e];
        aw[k][e] = fmaf(dy[k][e], xh[k][e], aw[k][e]);
        if (g.w) dy[k][e] *= w[e];
        const float own = c.owns(e) ? dy[k][e] : 0.f;
        s1 += own;
        s2 = fmaf(own, xh[k][e], s2);
      }
    }
    const float2 sum = row_sums<WPR>(s1, s2, s_red, turn++);
    s1 = sum.x * inv_d;
    s2 = sum.y * inv_d;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const Cols<WPR> c(k, t, g.d);
      if (!c.any()) continue;
      typename Vec8<TX>::type res;
      if (g.dres) res = Vec8<TX>::load((const TX*)g.dres + r * g.d + c.base);
      float o[kV];
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        o[e] = rstd * (dy[k][e] - s1 - xh[k][e] * s2);
        if (g.dres) o[e] += (float)res[e];
      }
      Vec8<TX>::store((TX*)g.dx + r * g.d + c.base, o);
    }
  }
  if (!g.part) return;
  float* part = g.part + (int64_t)blockIdx.x * 2 * g.d;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    if (WPR == 1 && q) __syncthreads();
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const Cols<WPR> c(k, t, g.d);
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (c.owns(e)) {
          const float v = q ? ab[k][e] : aw[k][e];
          if constexpr (WPR == 1)
            s_acc[wave][c.base + e] = v;
          else
            part[q * g.d + c.base + e] = v;
        }
    }
    if constexpr (WPR == 1) {
      __syncthreads();
      for (int64_t c = threadIdx.x; c < g.d; c += 64 * kWaves)
        part[q * g.d + c] = s_acc[0][c] + s_acc[1][c] + s_acc[2][c] + s_acc[3][c];
    }
  }
}

// Rows of any other width (below kV, or more than a workgroup holds), a
// workgroup each, read again for every pass. A lane's share of a wide row has no
// bound, so what it adds up over it is held in 64 bits: float32 sums of squares
// over 2^26 columns left rstd off by 3e-5.
template <typename TX, typename TY>
__global__ __launch_bounds__(64 * kWaves) void norm_fwd_any_kernel(const NormArgs g) {
  __shared__ float2 s_red[2][4];
  const int64_t r = blockIdx.x;
  const TX* row = (const TX*)g.x + r * g.x_ld;
  double s = 0.0;
  for (int64_t c = threadIdx.x * kV; c < g.d; c += 64 * kWaves * kV) {
    float v[kV];
    load8(row, c, g.d, v);
    float p = 0.f;
#pragma unroll
    for (int e = 0; e < kV; ++e) p += v[e];
    s += (double)p;
  }
  const float mean = row_sum<kWaves>((float)s, s_red, 0) / (float)g.d;
  s = 0.0;
  for (int64_t c = threadIdx.x * kV; c < g.d; c += 64 * kWaves * kV) {
    float v[kV];
    load8(row, c, g.d, v);
    float p = 0.f;
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      const float u = c + e < g.d ? v[e] - mean : 0.f;
      p = fmaf(u, u, p);
    }
    s += (double)p;
  }
  const float rstd = 1.f / sqrtf(row_sum<kWaves>((float)s, s_red, 1) / (float)g.d + g.eps);
  for (int64_t c = threadIdx.x * kV; c < g.d; c += 64 * kWaves * kV) {
    float v[kV], w[kV], b[kV];
    load8(row, c, g.d, v);
    if (g.w) load8(g.w, c, g.d, w);
    if (g.b) load8(g.b, c, g.d, b);
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      float o = (v[e] - mean) * rstd;
      if (g.w) o *= w[e];
      if (g.b) o += b[e];
      v[e] = o;
    }
    store8((TY*)g.y + r * g.d, c, g.d, v);
  }
  if (threadIdx.x == 0 && g.mean) {
    g.mean[r] = mean;
    g.rstd[r] = rstd;
  }
}

template <typename TX, typename TY>
__global__ __launch_bounds__(64 * kWaves) void norm_dx_any_kernel(const NormArgs g) {
  __shared__ float2 s_red[2][4];
  const int64_t r = blockIdx.x;
  const float mean = g.mean[r], rstd = g.rstd[r];
  const TX* x = (const TX*)g.x + r * g.x_ld;
  const TY* dy = (const TY*)g.dy + r * g.dy_ld;
  double t1 = 0.0, t2 = 0.0;
  float s1 = 0.f, s2 = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t c = threadIdx.x * kV; c < g.d; c += 64 * kWaves * kV) {
      float xv[kV], gv[kV], w[kV], res[kV];
      load8(x, c, g.d, xv);
      load8(dy, c, g.d, gv);
      if (g.w) load8(g.w, c, g.d, w);
      if (pass && g.dres) load8((const TX*)g.dres + r * g.d, c, g.d, res);
      float p1 = 0.f, p2 = 0.f;
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        const float xh = (xv[e] - mean) * rstd;
        if (g.w) gv[e] *= w[e];
        if (pass == 0) {
          p1 += gv[e];
          p2 = fmaf(gv[e], xh, p2);
        } else {
          gv[e] = rstd * (gv[e] - s1 - xh * s2);
          if (g.dres) gv[e] += res[e];
        }
      }
      t1 += (double)p1;
      t2 += (double)p2;
      if (pass) store8((TX*)g.dx + r * g.d, c, g.d, gv);
    }
    if (pass == 0) {
      const float2 sum = row_sums<kWaves>((float)t1, (float)t2, s_red, 0);
      s1 = sum.x / (float)g.d;
      s2 = sum.y / (float)g.d;
    }
  }
}

constexpr int kAnyRows = 4;  // rows that a lane below loads before the first is added

// dw and db terms of those widths: a workgroup takes `cols` columns (a power of
// two) by 256 / cols rows at once, rows gridDim.y times as many apart, in 64
// bits as above. 2^24 rows x 4 in bfloat16, the whole backward: 32 ms (140 with
// 256 columns a workgroup whatever the width, of which narrow rows used four).
template <typename TX, typename TY>
__global__ __launch_bounds__(64 * kWaves) void norm_cols_any_kernel(const NormArgs g, int cols) {
  __shared__ double s_acc[2][64 * kWaves];
  const int t = threadIdx.x, per = 64 * kWaves / cols;
  const int64_t c = (int64_t)blockIdx.x * cols + (t & (cols - 1));
  double aw = 0.0, ab = 0.0;
  constexpr int kU = kAnyRows;  // added in float32 among themselves
  const int64_t hop = (int64_t)gridDim.y * per;
  if (c < g.d)
    for (int64_t r0 = (int64_t)blockIdx.y * per + t / cols; r0 < g.rows; r0 += kU * hop) {
      float dy[kU], xh[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t r = r0 + u * hop < g.rows ? r0 + u * hop : r0;
        dy[u] = (float)((const TY*)g.dy)[r * g.dy_ld + c];
        xh[u] = ((float)((const TX*)g.x)[r * g.x_ld + c] - g.mean[r]) * g.rstd[r];
      }
      float pw = 0.f, pb = 0.f;
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (r0 + u * hop < g.rows) {
          pw = fmaf(dy[u], xh[u], pw);
          pb += dy[u];
        }
      aw += (double)pw;
      ab += (double)pb;
    }
  // the rows' lanes join in halves
  s_acc[0][t] = aw;
  s_acc[1][t] = ab;
  for (int h = per / 2; h >= 1; h >>= 1) {
    __syncthreads();
    if (t < h * cols) {
      s_acc[0][t] += s_acc[0][t + h * cols];
      s_acc[1][t] += s_acc[1][t + h * cols];
    }
  }
  if (t < cols && c < g.d) {
    float* part = g.part + (int64_t)blockIdx.y * 2 * g.d;
    part[c] = (float)s_acc[0][t];
    part[g.d + c] = (float)s_acc[1][t];
  }
}

// dw[c], db[c] = the sums over n rows of part [n][2][d], in a fixed order and in
// 64 bits (n grows with the rows): 32 columns a workgroup at a time, each of 32
// groups of lanes adds every 32nd row.
__global__ __launch_bounds__(1024) void norm_fold_kernel(const float* __restrict__ part, int n, int64_t d,
                                                         float* __restrict__ dw, float* __restrict__ db) {
  __shared__ double s[32][33];
  const int col = threadIdx.x & 31, q = threadIdx.x >> 5;
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < 2 * d; c0 += (int64_t)gridDim.x * 32) {
    const int64_t c = c0 + col;
    double acc = 0.0;
    if (c < 2 * d) {
      constexpr int kU = 8;  // rows loaded before the first is added
      int i = q;
      for (; i + (kU - 1) * 32 < n; i += kU * 32) {
        float v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) v[u] = part[(int64_t)(i + u * 32) * 2 * d + c];
#pragma unroll
        for (int u = 0; u < kU; ++u) acc += v[u];
      }
      for (; i < n; i += 32) acc += part[(int64_t)i * 2 * d + c];
    }
    s[q][col] = acc;
    __syncthreads();
    if (q == 0 && c < 2 * d) {
      double t = 0.0;
#pragma unroll
      for (int w = 0; w < 32; ++w) t += s[w][col];
      if (c < d) {
        if (dw) dw[c] = (float)t;
      } else if (db) {
        db[c - d] = (float)t;
      }
    }
    __syncthreads();
  }
}

// dst[r][c] = src[r][c] for c < cols, 0 for cols <= c < dst_ld (a multiple of
// 8): rows of 16-bit values brought to an aligned stride.
__global__ __launch_bounds__(256) void pack_rows_kernel(const uint16_t* __restrict__ src, int64_t src_ld, int64_t rows,
                                                        int64_t cols, uint16_t* __restrict__ dst, int64_t dst_ld) {
  typedef UserVec<uint16_t, 8, 2>::type u8v;
  const int64_t per = dst_ld / 8, n = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = (i - r * per) * 8;
    const uint16_t* p = src + r * src_ld + c;
    u8v v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c + 8 <= cols)
      v = *reinterpret_cast<const u8v*>(p);
    else
      for (int e = 0; c + e < cols; ++e) v[e] = p[e];
    *reinterpret_cast<u8v*>(dst + r * dst_ld + c) = v;
  }
}

// ------------------------------------------------------------------ host side

bool dt_ok(int dt) { return dt == NAJU_DTYPE_F32 || dt == NAJU_DTYPE_BF16 || dt == NAJU_DTYPE_F16; }

// Columns that WPR waves with G groups a lane hold.
constexpr int64_t held(int wpr, int G) { return (int64_t)wpr * G * 64 * kV; }
bool in_registers(int64_t d) { return d >= kV && d <= held(kWaves, 8); }

// Workgroups of the backward in registers: rows are taken in turn by 768 of them,
// three on a CU (65536 x 4096 bf16: 352 us; 369 with 512 of them, 422 with 1024,
// 377 with 2048; 16384 x 768: 26 us; 28, 31 and 35). With so many rows that a
// wave's float32 sums of dw and db would have more than kChain terms, by the
// next multiple of 768 that keeps to it: terms of one sign are then off by
// kChain 2^-24 at most.
constexpr int kBwdGrid = 768, kChain = 1024;
int64_t bwd_grid(int64_t rows, int64_t d) {
  const int64_t per = d <= held(1, 2) ? kWaves : 1;
  const int64_t n = (rows + per - 1) / per;
  if (n <= kBwdGrid) return n;
  return (n + kBwdGrid * kChain - 1) / (kBwdGrid * kChain) * kBwdGrid;
}
// Columns that a workgroup of norm_cols_any_kernel takes, and its row slices:
// narrow rows are one workgroup wide, so that it takes many slices to fill the CUs.
int any_cols(int64_t d) { return d > 4 ? (d < kV ? kV : 64 * kWaves) : d > 2 ? 4 : (int)d; }
int64_t any_slices(int64_t rows, int64_t d) {
  const int64_t per = 64 * kWaves / any_cols(d) * kAnyRows, most = d < kV ? 1024 : 64;
  const int64_t n = (rows + per - 1) / per;
  return n < most ? n : most;
}

// Rows of one launch of a workgroup a row: a launch has fewer than 2^32 threads.
constexpr int64_t kLaunchRows = 1 << 23;

// From row r on, as many as one launch takes.
template <typename TX, typename TY>
NormArgs rows_from(NormArgs g, int64_t r) {
  g.rows = g.rows - r < kLaunchRows ? g.rows - r : kLaunchRows;
  g.x = (const TX*)g.x + r * g.x_ld;
  if (g.y) g.y = (TY*)g.y + r * g.d;
  if (g.mean) g.mean += r;
  if (g.rstd) g.rstd += r;
  if (g.dy) g.dy = (const TY*)g.dy + r * g.dy_ld;
  if (g.dres) g.dres = (const TX*)g.dres + r * g.d;
  if (g.dx) g.dx = (TX*)g.dx + r * g.d;
  return g;
}

template <typename TX, typename TY>
void fwd_launch(const NormArgs& g, hipStream_t st) {
  if (g.rows > kLaunchRows) {
    for (int64_t r = 0; r < g.rows; r += kLaunchRows) fwd_launch<TX, TY>(rows_from<TX, TY>(g, r), st);
    return;
  }
  const dim3 blk(64 * kWaves), by_wave((unsigned)((g.rows + kWaves - 1) / kWaves)), by_row((unsigned)g.rows);
  if (!in_registers(g.d))
    norm_fwd_any_kernel<TX, TY><<<by_row, blk, 0, st>>>(g);
  else if (g.d <= held(1, 1))
    norm_fwd_kernel<TX, TY, 1, 1><<<by_wave, blk, 0, st>>>(g);
  else if (g.d <= held(1, 2))
    norm_fwd_kernel<TX, TY, 1, 2><<<by_wave, blk, 0, st>>>(g);
  else if (g.d <= held(1, 4))
    norm_fwd_kernel<TX, TY, 1, 4><<<by_wave, blk, 0, st>>>(g);
  else if (g.d <= held(kWaves, 2))
    norm_fwd_kernel<TX, TY, kWaves, 2><<<by_row, blk, 0, st>>>(g);
  else if (g.d <= held(kWaves, 4))
    norm_fwd_kernel<TX, TY, kWaves, 4><<<by_row, blk, 0, st>>>(g);
  else
    norm_fwd_kernel<TX, TY, kWaves, 8><<<by_row, blk, 0, st>>>(g);
}

// A row by one wave to 1024 columns, by a workgroup above (32768 rows, bf16: 1536
// columns 112 and 73 us, 2048 135 and 84; float32 142 and 125, 175 and 162): more
// registers a lane leave too few waves a CU. The forward, which holds half as
// much, keeps to one wave up to 2048 (37 us there in bf16, 52 by a workgroup).
template <typename TX, typename TY>
void bwd_launch(const NormArgs& g, float* dw, float* db, hipStream_t st) {
  const dim3 blk(64 * kWaves), grid((unsigned)bwd_grid(g.rows, g.d));
  int64_t n = grid.x;
  if (!in_registers(g.d)) {
    for (int64_t r = 0; r < g.rows; r += kLaunchRows) {
      const NormArgs p = rows_from<TX, TY>(g, r);
      norm_dx_any_kernel<TX, TY><<<dim3((unsigned)p.rows), blk, 0, st>>>(p);
    }
    if (g.part) {
      const int cols = any_cols(g.d);
      n = any_slices(g.rows, g.d);
      norm_cols_any_kernel<TX, TY>
          <<<dim3((unsigned)((g.d + cols - 1) / cols), (unsigned)n), blk, 0, st>>>(g, cols);
    }
  } else if (g.d <= held(1, 1))
    norm_bwd_kernel<TX, TY, 1, 1><<<grid, blk, 0, st>>>(g);
  else if (g.d <= held(1, 2))
    norm_bwd_kernel<TX, TY, 1, 2><<<grid, blk, 0, st>>>(g);
  else if (g.d <= held(kWaves, 1))
    norm_bwd_kernel<TX, TY, kWaves, 1><<<grid, blk, 0, st>>>(g);
  else if (g.d <= held(kWaves, 2))
    norm_bwd_kernel<TX, TY, kWaves, 2><<<grid, blk, 0, st>>>(g);
  else if (g.d <= held(kWaves, 4))
    norm_bwd_kernel<TX, TY, kWaves, 4><<<grid, blk, 0, st>>>(g);
  else
    norm_bwd_kernel<TX, TY, kWaves, 8><<<grid, blk, 0, st>>>(g);
  if (g.part) {
    // (a launch has fewer than 2^32 threads: wider rows take turns)
    const int64_t folds = (2 * g.d + 31) / 32, most = 1 << 20;
    norm_fold_kernel<<<dim3((unsigned)(folds < most ? folds : most)), 1024, 0, st>>>(g.part, (int)n, g.d, dw, db);
  }
}

template <typename TX>
void fwd_dispatch(const NormArgs& g, int y_dt, hipStream_t st) {
  if (y_dt == NAJU_DTYPE_F32)
    fwd_launch<TX, float>(g, st);
  else if (y_dt == NAJU_DTYPE_BF16)
    fwd_launch<TX, bf16_t>(g, st);
  else
    fwd_launch<TX, f16_t>(g, st);
}
template <typename TX>
void bwd_dispatch(const NormArgs& g, int dy_dt, float* dw, float* db, hipStream_t st) {
  if (dy_dt == NAJU_DTYPE_F32)
    bwd_launch<TX, float>(g, dw, db, st);
  else if (dy_dt == NAJU_DTYPE_BF16)
    bwd_launch<TX, bf16_t>(g, dw, db, st);
  else
    bwd_launch<TX, f16_t>(g, dw, db, st);
}

int launched() {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mixer_fail(NAJU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
  return NAJU_OK;
}

int check_norm(int64_t rows, int64_t d, int64_t ld, int64_t ld2, int x_dt, int y_dt) {
  if (rows < 0 || d < 1) return mixer_fail(NAJU_ERR_INVALID, "n_rows must be >= 0 and d positive");
  if (ld < d || ld2 < d) return mixer_fail(NAJU_ERR_INVALID, "row strides must be >= d (%lld)", (long long)d);
  if (!dt_ok(x_dt) || !dt_ok(y_dt)) return mixer_fail(NAJU_ERR_INVALID, "unknown dtype code");
  if (rows > 0x7fffffff || d > (1 << 30)) return mixer_fail(NAJU_ERR_UNSUPPORTED, "shape too large");
  return NAJU_OK;
}

}  // namespace
}  // namespace naju_detail

using namespace naju_detail;

extern "C" {

int naju_layernorm_fwd(const void* x, int64_t x_ld, const float* w, const float* b, float eps, void* y, float* mean,
                       float* rstd, int64_t n_rows, int64_t d, int x_dtype, int y_dtype, void* stream) {
  mixer_clear();
  int rc = check_norm(n_rows, d, x_ld, d, x_dtype, y_dtype);
  if (rc) return rc;
  if (!mean != !rstd) return mixer_fail(NAJU_ERR_INVALID, "mean and rstd come together");
  if (n_rows == 0) return NAJU_OK;
  if (!x || !y) return mixer_fail(NAJU_ERR_INVALID, "null pointer (x and y are required)");
  NormArgs g = {};
  g.x = x;
  g.x_ld = x_ld;
  g.w = w;
  g.b = b;
  g.eps = eps;
  g.y = y;
  g.mean = mean;
  g.rstd = rstd;
  g.rows = n_rows;
  g.d = d;
  hipStream_t st = (hipStream_t)stream;
  if (x_dtype == NAJU_DTYPE_F32)
    fwd_dispatch<float>(g, y_dtype, st);
  else if (x_dtype == NAJU_DTYPE_BF16)
    fwd_dispatch<bf16_t>(g, y_dtype, st);
  else
    fwd_dispatch<f16_t>(g, y_dtype, st);
  return launched();
}

size_t naju_layernorm_workspace_bytes(int64_t n_rows, int64_t d) {
  if (n_rows < 0 || d < 1) return 0;
  const int64_t n = in_registers(d) ? bwd_grid(n_rows, d) : any_slices(n_rows, d);
  return (size_t)(n * 2 * d) * sizeof(float) + 256;
}

int naju_layernorm_bwd(const void* x, int64_t x_ld, const float* w, const float* mean, const float* rstd,
                       const void* dy, int64_t dy_ld, const void* dres, void* dx, float* dw, float* db, int64_t n_rows,
                       int64_t d, int x_dtype, int dy_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  mixer_clear();
  int rc = check_norm(n_rows, d, x_ld, dy_ld, x_dtype, dy_dtype);
  if (rc) return rc;
  if (n_rows == 0) return NAJU_OK;
  if (!x || !mean || !rstd || !dy || !dx)
    return mixer_fail(NAJU_ERR_INVALID, "null pointer (x, mean, rstd, dy and dx are required)");
  const bool sums = dw || db;
  if (sums && (!workspace || workspace_bytes < naju_layernorm_workspace_bytes(n_rows, d)))
    return mixer_fail(NAJU_ERR_WORKSPACE, "workspace of %zu bytes needed", naju_layernorm_workspace_bytes(n_rows, d));
  NormArgs g = {};
  g.x = x;
  g.x_ld = x_ld;
  g.w = w;
  g.mean = (float*)mean;
  g.rstd = (float*)rstd;
  g.dy = dy;
  g.dy_ld = dy_ld;
  g.dres = dres;
  g.dx = dx;
  g.part = sums ? (float*)workspace : nullptr;
  g.rows = n_rows;
  g.d = d;
  hipStream_t st = (hipStream_t)stream;
  if (x_dtype == NAJU_DTYPE_F32)
    bwd_dispatch<float>(g, dy_dtype, dw, db, st);
  else if (x_dtype == NAJU_DTYPE_BF16)
    bwd_dispatch<bf16_t>(g, dy_dtype, dw, db, st);
  else
    bwd_dispatch<f16_t>(g, dy_dtype, dw, db, st);
  return launched();
}

int naju_pack_rows(const void* src, int64_t src_ld, int64_t n_rows, int64_t n_cols, void* dst, int64_t dst_ld,
                   void* stream) {
  mixer_clear();
  if (n_rows < 0 || n_cols < 0 || src_ld < n_cols || dst_ld < n_cols || dst_ld % 8)
    return mixer_fail(NAJU_ERR_INVALID, "row strides must be >= n_cols, dst_ld a multiple of 8");
  if (n_rows == 0 || dst_ld == 0) return NAJU_OK;
  if (!src || !dst) return mixer_fail(NAJU_ERR_INVALID, "null pointer (src and dst are required)");
  if (n_rows > (1ll << 40) / dst_ld) return mixer_fail(NAJU_ERR_UNSUPPORTED, "shape too large");
  const int64_t wgs = (n_rows * (dst_ld / 8) + 255) / 256;
  pack_rows_kernel<<<dim3((unsigned)(wgs < 4096 ? wgs : 4096)), 256, 0, (hipStream_t)stream>>>(
      (const uint16_t*)src, src_ld, n_rows, n_cols, (uint16_t*)dst, dst_ld);
  return launched();
}

}  // extern "C"
