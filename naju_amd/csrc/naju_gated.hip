// naju_gated.hip -- the gated feed-forward product h = act(x Wg^T) * (x Wu^T)
// and its gradients on MI355X (gfx950), behind the C ABI of
// include/naju_mixer.h.
//
// Forward: one tile kernel whose n operand alternates 32 rows of Wg with the
// same 32 rows of Wu, so that a lane's accumulators hold a gate and its up
// projection in corresponding registers: the activation and the product are
// done on them, and only h is written.
//
// Backward: nothing of size n_rows x f is kept from the forward. The same tile
// kernel forms both projections again and, from dh, writes
//   dg = dh * u * act'(g),   du = dh * act(g)
// in 16 bits (each rounded once from float32, as the gradients of 16-bit
// projections are) side by side into the workspace; then
//   dx  = dg Wg + du Wu            one product over both halves' k
//   dWg = dg^T x, dWu = du^T x     one product, the halves' rows to two outputs
// (gemm_out.h).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "gemm_few.h"
#include "gemm_out.h"
#include "naju_mixer.h"
#include "naju_scan.h"

namespace naju_detail {
int mixer_fail(int code, const char* fmt, ...);
void mixer_clear();

namespace {

// act(g) and act'(g)
template <int ACT>
__device__ __forceinline__ float act_fwd(float g) {
  if constexpr (ACT == NAJU_ACT_SILU) return g * sigm(g);
  return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
}
template <int ACT>
__device__ __forceinline__ void act_bwd(float g, float& a, float& da) {
  if constexpr (ACT == NAJU_ACT_SILU) {
    const float s = sigm(g);
    a = g * s;
    da = s * fmaf(g, 1.f - s, 1.f);
  } else {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    da = fmaf(g * 0.39894228040143268f, __builtin_amdgcn_exp2f(g * g * -0.72134752044448170f), cdf);
  }
}

struct GatedArgs {
  const char* x;
  const char* wg;
  const char* wu;
  int64_t x_ld, w_ld;  // bytes
  int64_t m, d, f;
  void* h;        // forward: [m][f]
  int64_t h_ld;   // elements
  const void* dh; // backward: [m][f]
  int64_t dh_ld;  // elements
  void* dgu;      // backward: [m][2 fp]: dg in columns [0, fp), du after them, zeros from f to fp
  int64_t fp;
};

template <typename T, typename C, int ACT, bool BWD>
__global__ __launch_bounds__(C::kThreads, 2) void gated_kernel(const GatedArgs g, int nm, int nn) {
  static_assert(C::TN == 4, "a wave's 64 columns are 32 gates and their 32 up projections");
  NAJU_GEMM_LDS(C);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int steps = (int)((g.d + kBK - 1) / kBK);
  TilePipe<T, C, kAlongK, kAlongK, true> pipe;
  int64_t m0 = 0, f0 = 0;
  const char *xb = nullptr, *gb = nullptr;
  const int64_t to_up = g.wu - g.wg;
  auto a_at = [&](int s) { return Step{xb + (int64_t)s * (kBK * 2), g.d - (int64_t)s * kBK, 0}; };
  auto b_at = [&](int s) { return Step{gb + (int64_t)s * (kBK * 2), g.d - (int64_t)s * kBK, to_up}; };
  auto begin = [&](int id) __attribute__((always_inline)) {
    int bm, bn;
    tile_of(id, nm, nn, bm, bn);
    m0 = (int64_t)bm * C::BM;
    f0 = (int64_t)bn * (C::BN / 2);
    const int ma = (int)(g.m - 1 - m0 < C::BM ? g.m - 1 - m0 : C::BM);
    const int fa = (int)(g.f - 1 - f0 < C::BN ? g.f - 1 - f0 : C::BN);
    xb = g.x + m0 * g.x_ld;
    gb = g.wg + f0 * g.w_ld;
    pipe.init((uint32_t)g.x_ld, (uint32_t)g.w_ld, [&](int r) { return r < ma ? r : ma; },
              [&](int r) {
                // rows 64 w + 0..31 are gates 32 w ..., rows 64 w + 32..63 their up projections
                const int f = (r >> 6) * 32 + (wide_row(r) & 31);
                return f < fa ? f : fa;
              });
    pipe.start(s_steps, steps, a_at, b_at);
  };
  int id = blockIdx.x;
  begin(id);
  for (;;) {
    acc_t acc[C::TM][C::TN];
    pipe.run(acc, s_steps, steps, a_at, b_at);
    const int64_t mw = m0 + (wave / C::WN) * C::TM * 16 + (lane & 15);
    const int64_t f = f0 + (wave % C::WN) * 32 + 8 * (lane >> 4);
    const int64_t left = g.f - f;
    id += gridDim.x;
    const bool more = id < nm * nn;
    if (more) begin(id);
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      const int64_t m = mw + i * 16;
      if (m >= g.m) continue;
      if constexpr (!BWD) {
        if (left <= 0) continue;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = act_fwd<ACT>(acc[i][e >> 2][e & 3]) * acc[i][(e >> 2) + 2][e & 3];
        store_row((T*)g.h + m * g.h_ld + f, o, left);
      } else {
        if (f >= g.fp) continue;
        float dh[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, og[8], ou[8];
        if (left > 0) load_row((const T*)g.dh + m * g.dh_ld + f, dh, left);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float a, da;
          act_bwd<ACT>(acc[i][e >> 2][e & 3], a, da);
          og[e] = e < left ? dh[e] * acc[i][(e >> 2) + 2][e & 3] * da : 0.f;
          ou[e] = e < left ? dh[e] * a : 0.f;
        }
        T* row = (T*)g.dgu + m * 2 * g.fp + f;
        store_row(row, og, 8);
        store_row(row + g.fp, ou, 8);
      }
    }
    if (!more) break;
  }
}

// Forward for at most 16 MT rows: 16 gates and their 16 up projections a
// workgroup.
template <typename T, int ACT, int MT>
__global__ __launch_bounds__(512) void gated_few_kernel(const GatedArgs g) {
  typedef FewProduct<T, 2, MT, 8> P;
  __shared__ float s[P::kFloats];
  const int64_t f0 = (int64_t)blockIdx.x * 16;
  P::run(
      s, g.d, [&](int r) { return g.x + (r < g.m ? r : g.m - 1) * g.x_ld; },
      [&](int r) {
        const int64_t f = f0 + (r & 15) < g.f ? f0 + (r & 15) : g.f - 1;
        return (r < 16 ? g.wg : g.wu) + f * g.w_ld;
      });
  for (int e = threadIdx.x; e < 16 * P::M; e += P::kThreads) {
    const int m = e >> 4, f = e & 15;
    if (m < g.m && f0 + f < g.f)
      ((T*)g.h)[m * g.h_ld + f0 + f] = (T)(act_fwd<ACT>(s[f * P::M + m]) * s[(16 + f) * P::M + m]);
  }
}

template <typename T, int ACT, bool BWD>
void gated_launch(const GatedArgs& g, hipStream_t st) {
  // Few rows: bound by the latency of the weights' loads. Here and on the tiles
  // below, cold weights, d = 768 / 2048 / 8192: 16 rows, f = 1024 4.5 / 7.8 / 27.8 and
  // 9.2 / 19.4 / 97.9 us, f = 8192 8.2 / 16.9 / 60.9 and 12.9 / 29.7 / 107, f = 28672 22.9 /
  // 56.8 / 212 and 24.6 / 58.1 / 222, f = 65536 (768 / 2048) 47.4 / 124 and 49.1 / 132; 32
  // rows, f = 8192 9.6 / 20.6 / 74.6 and 13.3 / 29.9 / 108, f = 16384 16.6 / 39.9 / 151 and
  // 14.9 / 34.3 / 136; 64 rows, f = 4096 8.6 / 16.2 / 54.9 and 12.9 / 28.9 / 102, f = 5504
  // 14.6 / 28.9 / 104 and 13.3 / 29.5 / 106.
  if (!BWD && (g.m <= 16 || (g.m <= 32 && g.f <= 8192) || (g.m <= 64 && g.f <= 4096))) {
    const unsigned grid = (unsigned)ceil_div(g.f, 16);
    if (g.m <= 16)
      gated_few_kernel<T, ACT, 1><<<grid, 512, 0, st>>>(g);
    else if (g.m <= 32)
      gated_few_kernel<T, ACT, 2><<<grid, 512, 0, st>>>(g);
    else
      gated_few_kernel<T, ACT, 4><<<grid, 512, 0, st>>>(g);
    return;
  }
  // backward tiles also cover the zero columns up to fp
  const int64_t f = BWD ? g.fp : g.f;
  const int64_t tl = ceil_div(g.m, TileL::BM) * ceil_div(f, TileL::BN / 2);
  // the large tile where the small ones, two a CU, would need a second round. Both
  // measured over 48 to 512 large tiles, d = 256, 768 and 2048 (2032 rows, d = 768;
  // large and small): forward 96 tiles 20.0 and 16.0 us, 128 20.3 and 18.3, 144 20.5
  // and 23.6, 256 26.3 and 38.1, 512 52.1 and 71.1; backward 128 27.8 and 23.8, 144
  // 27.4 and 32.1, 256 31.6 and 41.0, 512 64.0 and 90.6. The rule loses where the
  // large tiles have just begun a second round themselves, 257 to about 300 of them:
  // at d = 768 up to 9% (288 tiles of 4080 rows backward 52.5 and 48.3), at d = 2048 up
  // to 4%, at d = 256 up to 19%.
  if (tl > kCUs / 2) {
    const int nm = (int)ceil_div(g.m, TileL::BM), nn = (int)ceil_div(f, TileL::BN / 2);
    gated_kernel<T, TileL, ACT, BWD><<<tile_grid<TileL>(nm * nn), TileL::kThreads, 0, st>>>(g, nm, nn);
  } else {
    const int nm = (int)ceil_div(g.m, TileS::BM), nn = (int)ceil_div(f, TileS::BN / 2);
    gated_kernel<T, TileS, ACT, BWD><<<tile_grid<TileS>(nm * nn), TileS::kThreads, 0, st>>>(g, nm, nn);
  }
}

template <bool BWD>
void gated_dispatch(const GatedArgs& g, int act, int dtype, hipStream_t st) {
  if (dtype == NAJU_DTYPE_BF16) {
    if (act == NAJU_ACT_SILU)
      gated_launch<bf16_t, NAJU_ACT_SILU, BWD>(g, st);
    else
      gated_launch<bf16_t, NAJU_ACT_GELU, BWD>(g, st);
  } else {
    if (act == NAJU_ACT_SILU)
      gated_launch<f16_t, NAJU_ACT_SILU, BWD>(g, st);
    else
      gated_launch<f16_t, NAJU_ACT_GELU, BWD>(g, st);
  }
}

template <typename T>
void weight_grad_launch(const GemmOut& g, const GemmPlan& p, int dw_dtype, hipStream_t st) {
  if (dw_dtype == NAJU_DTYPE_F32)
    gemm_out_launch<T, float, kAlongMN>(g, p, st);
  else
    gemm_out_launch<T, T, kAlongMN>(g, p, st);
}

int launched() {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return mixer_fail(NAJU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
  return NAJU_OK;
}

int check_gated(const void* x, int64_t x_ld, const void* wg, const void* wu, int64_t w_ld, int64_t n_rows, int64_t d,
                int64_t f, int act, int dtype) {
  if (n_rows < 0 || d < 1 || f < 1) return mixer_fail(NAJU_ERR_INVALID, "n_rows must be >= 0, d and f positive");
  if (act != NAJU_ACT_SILU && act != NAJU_ACT_GELU) return mixer_fail(NAJU_ERR_INVALID, "unknown activation %d", act);
  if (dtype != NAJU_DTYPE_BF16 && dtype != NAJU_DTYPE_F16)
    return mixer_fail(NAJU_ERR_UNSUPPORTED, "the gated product serves bf16 and f16");
  // f too: the backward's rows of both projections' gradients are 2 f elements,
  // and the offsets within a tile (255 rows) are 32 bits
  if (n_rows > (1ll << 30) || d > (1 << 21) || f > (1 << 21) || x_ld > (1 << 21) || w_ld > (1 << 21) ||
      !tiles_fit(n_rows, f) || !tiles_fit(2 * f, d))
    return mixer_fail(NAJU_ERR_UNSUPPORTED, "shape too large (d, f and row strides up to 2^21 elements)");
  const int64_t d8 = round_up(d, 8);
  if (x_ld < d8 || w_ld < d8 || x_ld % 8 || w_ld % 8)
    return mixer_fail(NAJU_ERR_INVALID, "row strides must be multiples of 8, at least d rounded up to 8");
  if (n_rows == 0) return NAJU_OK;
  if (!x || !wg || !wu) return mixer_fail(NAJU_ERR_INVALID, "null pointer (x and both weights are required)");
  if (((uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu) & 15)
    return mixer_fail(NAJU_ERR_INVALID, "x and the weights must be 16-byte aligned");
  return NAJU_OK;
}

// The backward's workspace: dgu, then the split sums of dx and of dW.
struct GatedBwdPlan {
  int64_t fp;
  GemmPlan dx, dw;
  size_t o_dx, o_dw, total;
};
GatedBwdPlan gated_bwd_plan(int64_t m, int64_t d, int64_t f) {
  GatedBwdPlan p;
  p.fp = round_up(f, kBK);  // dx's product finds du at a step of k
  p.dx = gemm_plan(m, d, f, f);
  p.dw = gemm_plan(2 * p.fp, d, m, 0);
  p.o_dx = (size_t)round_up(m * 2 * p.fp * 2, 256);
  // dx is complete before dW's product starts: one region serves both
  p.o_dw = p.o_dx;
  const size_t a = gemm_part_bytes(p.dx, m, d), b = gemm_part_bytes(p.dw, 2 * p.fp, d);
  p.total = p.o_dx + (a > b ? a : b) + 256;
  return p;
}

}  // namespace
}  // namespace naju_detail

using namespace naju_detail;

extern "C" {

int naju_gated_fwd(const void* x, int64_t x_ld, const void* w_gate, const void* w_up, int64_t w_ld, void* h,
                   int64_t h_ld, int64_t n_rows, int64_t d, int64_t f, int act, int dtype, void* stream) {
  mixer_clear();
  int rc = check_gated(x, x_ld, w_gate, w_up, w_ld, n_rows, d, f, act, dtype);
  if (rc) return rc;
  if (h_ld < f) return mixer_fail(NAJU_ERR_INVALID, "h_ld (%lld) must be >= f (%lld)", (long long)h_ld, (long long)f);
  if (n_rows == 0) return NAJU_OK;
  if (!h) return mixer_fail(NAJU_ERR_INVALID, "null pointer (h is required)");
  GatedArgs g = {};
  g.x = (const char*)x;
  g.wg = (const char*)w_gate;
  g.wu = (const char*)w_up;
  g.x_ld = x_ld * 2;
  g.w_ld = w_ld * 2;
  g.m = n_rows;
  g.d = d;
  g.f = f;
  g.h = h;
  g.h_ld = h_ld;
  gated_dispatch<false>(g, act, dtype, (hipStream_t)stream);
  return launched();
}

size_t naju_gated_workspace_bytes(int64_t n_rows, int64_t d, int64_t f) {
  if (n_rows < 0 || d < 1 || f < 1) return 0;
  return gated_bwd_plan(n_rows, d, f).total;
}

int naju_gated_bwd(const void* x, int64_t x_ld, const void* w_gate, const void* w_up, int64_t w_ld, const void* dh,
                   int64_t dh_ld, void* dx, void* dw_gate, void* dw_up, int64_t n_rows, int64_t d, int64_t f, int act,
                   int dtype, int dw_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  mixer_clear();
  int rc = check_gated(x, x_ld, w_gate, w_up, w_ld, n_rows, d, f, act, dtype);
  if (rc) return rc;
  if (dh_ld < f)
    return mixer_fail(NAJU_ERR_INVALID, "dh_ld (%lld) must be >= f (%lld)", (long long)dh_ld, (long long)f);
  if (dw_dtype != dtype && dw_dtype != NAJU_DTYPE_F32)
    return mixer_fail(NAJU_ERR_INVALID, "dw_dtype must be the operands' dtype or f32");
  if (!dw_gate != !dw_up) return mixer_fail(NAJU_ERR_INVALID, "dw_gate and dw_up come together");
  hipStream_t st = (hipStream_t)stream;
  if (n_rows == 0) return NAJU_OK;
  if (!dh) return mixer_fail(NAJU_ERR_INVALID, "null pointer (dh is required)");
  const GatedBwdPlan p = gated_bwd_plan(n_rows, d, f);
  if (!workspace || workspace_bytes < p.total)
    return mixer_fail(NAJU_ERR_WORKSPACE, "workspace of %zu bytes needed", p.total);
  if ((uintptr_t)workspace & 255) return mixer_fail(NAJU_ERR_INVALID, "workspace must be 256-byte aligned");
  GatedArgs g = {};
  g.x = (const char*)x;
  g.wg = (const char*)w_gate;
  g.wu = (const char*)w_up;
  g.x_ld = x_ld * 2;
  g.w_ld = w_ld * 2;
  g.m = n_rows;
  g.d = d;
  g.f = f;
  g.dh = dh;
  g.dh_ld = dh_ld;
  g.dgu = workspace;
  g.fp = p.fp;
  gated_dispatch<true>(g, act, dtype, st);
  if ((rc = launched())) return rc;
  if (dx) {
    GemmOut o = {};
    o.a = (const char*)workspace;
    o.lda = 2 * p.fp * 2;
    o.b[0] = g.wg;
    o.b[1] = g.wu;
    o.ldb = g.w_ld;
    o.k_first = o.k_second = f;
    o.m = n_rows;
    o.n = d;
    o.part = (float*)((char*)workspace + p.o_dx);
    o.out[0] = dx;
    o.ldo = d;
    o.m_half = o.out_rows = n_rows;
    if (dtype == NAJU_DTYPE_BF16)
      gemm_out_launch<bf16_t, bf16_t, kAlongK>(o, p.dx, st);
    else
      gemm_out_launch<f16_t, f16_t, kAlongK>(o, p.dx, st);
    if ((rc = launched())) return rc;
  }
  if (dw_gate) {
    GemmOut o = {};
    o.a = (const char*)workspace;
    o.lda = 2 * p.fp * 2;
    o.b[0] = o.b[1] = g.x;
    o.ldb = g.x_ld;
    o.k_first = n_rows;
    o.m = 2 * p.fp;
    o.n = d;
    o.part = (float*)((char*)workspace + p.o_dw);
    o.out[0] = dw_gate;
    o.out[1] = dw_up;
    o.ldo = d;
    o.m_half = p.fp;
    o.out_rows = f;
    if (dtype == NAJU_DTYPE_BF16)
      weight_grad_launch<bf16_t>(o, p.dw, dw_dtype, st);
    else
      weight_grad_launch<f16_t>(o, p.dw, dw_dtype, st);
    if ((rc = launched())) return rc;
  }
  return NAJU_OK;
}

}  // extern "C"
