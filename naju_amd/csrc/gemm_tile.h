// gemm_tile.h -- the 16-bit matrix-product tile that the gated feed-forward and
// the vocabulary-head kernels share (naju_gated.hip, naju_linear_xent.hip).
// Internal to the library.
//
// A workgroup forms a BM x BN tile of C[m][n] = sum_k A(m,k) B(n,k) in
// float32 registers. Each operand lies in memory in one of two ways:
//   kAlongK : rows of m (or n), k contiguous        (activations, weights of x W^T)
//   kAlongMN: rows of k, m (or n) contiguous        (weights of dy W, both of dy^T x)
// Either goes from memory to LDS without passing registers (16 bytes a lane),
// in steps of 32 k, three steps ahead of the products. LDS holds the step as
// it lies in memory, with the 16-byte pieces of a row permuted by an XOR of
// the row's number so that the lanes of one read fall on different banks;
// kAlongMN steps are read with the transposing LDS load.
//
// The products are v_mfma_f32_16x16x32 with the n operand as the instruction's
// rows: lane l then holds C[m = l % 16][n = 4 (l / 16) + r], four neighbouring
// n of one m, which the epilogues store as one vector and reduce over n mostly
// within the lane.
//
// What bounds it: 256 x 256 with eight waves of 128 x 64 reads 12 fragments of
// 1 KB from LDS for 32 products, which keeps LDS (128 bytes a clock) and the
// matrix cores about equally busy. Fragments of the next step are read behind
// the products that used their registers last, with one barrier a step: 8192^3 in
// bf16, random operands, at 1280 to 1340 TFLOP/s (least time of ten; 1140 to 1270 in
// the mean, at 1.6 GHz) in any of the three layouts, matrix cores 63 to 73% busy, no
// LDS bank conflicts (1160 with two steps of 64 k and the reads at the head of each,
// when this loop stood at 1290; a library product reached 1440 then).
// Four waves of 128 x 128 would read a third less, but the compiler moves
// their accumulators between register files in the loop (110 TFLOP/s).
//
// Bounds: rows past an operand's end are clamped to its last row (their
// products are discarded by the epilogues); k past the end reads as zero in
// both operands, through the buffer descriptor's range check.
#ifndef NAJU_GEMM_TILE_H
#define NAJU_GEMM_TILE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "scan_internal.h"

namespace naju_detail {
namespace {

typedef float acc_t __attribute__((ext_vector_type(4)));

enum Along { kAlongK, kAlongMN };
constexpr int kBK = 32;  // k of a step, and of one product

template <typename T>
struct Frag;
template <>
struct Frag<bf16_t> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ acc_t mma(v8 a, v8 b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<f16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ acc_t mma(v8 a, v8 b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// V neighbouring values of a caller's row, of which n exist, aligned to their
// elements and no more (see UserVec).
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&v)[V], int64_t n) {
  typedef typename UserVec<T, V, sizeof(T)>::type vec;
  if (n >= V) {
    vec o;
#pragma unroll
    for (int r = 0; r < V; ++r) o[r] = (T)v[r];
    *reinterpret_cast<vec*>(p) = o;
  } else {
#pragma unroll
    for (int r = 0; r < V; ++r)
      if (r < n) p[r] = (T)v[r];
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, float (&v)[V], int64_t n) {
  typedef typename UserVec<T, V, sizeof(T)>::type vec;
  if (n >= V) {
    const vec o = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] = (float)o[r];
  } else {
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] = r < n ? (float)p[r] : 0.f;
  }
}

// A step of one operand: its base address, and how many of its k exist (any
// number from kBK up means all). to_pair: the distance in bytes to a second
// operand whose rows alternate with the first's in the tile by 32 (the two
// weights of a gated product: a wave's 64 columns are then 32 of each).
struct Step {
  const char* base;
  int64_t k_left;
  int64_t to_pair;
};

// One operand of a tile: `rows` of the tile's R rows of m (or n) exist from
// `base` on. kAlongK: row r of the tile starts at base + r * ld. kAlongMN: k
// row j starts at base + j * ld and holds the tile's R columns. ld in bytes.
template <int R, int NW, Along AL>
struct Stage {
  static constexpr int kBytes = R * kBK * 2;
  static constexpr int kLoads = kBytes / 1024 / NW;  // wave loads of 1024 bytes, per wave
  static_assert(kLoads * NW * 1024 == kBytes, "tile rows must fill the waves' loads");
  static constexpr int kRowBytes = AL == kAlongK ? kBK * 2 : R * 2;
  static constexpr int kUnits = R / 16;  // 32-byte units of a kAlongMN row
  static_assert(kUnits % 8 == 0, "whole groups of eight units");

  uint32_t voff[kLoads];  // this lane's byte offset of each load from the step's base
  // the first k that each load of this lane covers within the step. Along k, or
  // where the waves' loads together are whole rows, that of the first load and a
  // constant for each after it; else (384 columns, eight waves: 10 2/3 rows) a
  // byte for each
  static constexpr bool kEven = AL == kAlongK || NW * 1024 % kRowBytes == 0;
  uint32_t kpos;
  __device__ __forceinline__ int k_of(int i) const {
    if constexpr (!kEven) return (int)(kpos >> (8 * i) & 255);
    return (int)kpos + (AL == kAlongK ? 0 : i * (NW * 1024 / kRowBytes));
  }

  // the XOR permutation of a kAlongMN row's 32-byte units: the 16 k rows that
  // one transposing read touches (k = 8 g + j, g and j below 4) differ in it, or
  // the eight of its halves where a row is not a whole number of 16 units
  static __device__ __forceinline__ int swz(int k) {
    return ((k & 3) | (((k >> 3) & 3) << 2)) & (kUnits % 16 == 0 ? 15 : 7);
  }

  // the same for a kAlongK row's 16-byte pieces: eight neighbouring rows of 64
  // bytes cover the banks
  static __device__ __forceinline__ int swz_k(int row) { return (row >> 1) & 3; }

  // map(r): the row (kAlongK) or column (kAlongMN, called for every eighth)
  // of the operand behind row r of the tile, relative to base, in bounds.
  template <typename Map>
  __device__ __forceinline__ void init(int wave, int lane, uint32_t ld, Map map) {
    static_assert(kEven || kLoads <= 4, "a byte of kpos for each load");
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int p = (i * NW + wave) * 1024 + lane * 16;
      const int row = p / kRowBytes, c = (p % kRowBytes) / 16;
      if constexpr (AL == kAlongK) {
        const int src = c ^ swz_k(row);
        voff[i] = (uint32_t)map(row) * ld + src * 16;
        kpos = src * 8;  // the same for every load: their rows differ by a multiple of 8
      } else {
        const int src = c ^ (swz(row) << 1);
        voff[i] = (uint32_t)row * ld + (uint32_t)map(src * 8) * 2;
        if constexpr (kEven) {
          if (i == 0) kpos = row;
        } else {
          kpos = (i == 0 ? 0 : kpos) | (uint32_t)row << (8 * i);
        }
      }
    }
  }

  // Starts the loads of one step, of which step.k_left k exist. kPair: rows of
  // the tile with bit 5 set come from the second operand (see Step).
  template <bool kPair>
  __device__ __forceinline__ void load(const Step& step, int wave, char* lds) const {
    constexpr int kRows = 1024 / kRowBytes;  // rows of one load
    static_assert(!kPair || (AL == kAlongK && 32 % kRows == 0), "a load's rows must lie in one operand");
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_one<kPair>(step, i, wave, lds);
  }
  template <bool kPair>
  __device__ __forceinline__ void load_one(const Step& step, int i, int wave, char* lds) const {
    constexpr uint32_t kRange = 0x7fffffffu;  // offsets past it read as zero
    constexpr int kRows = 1024 / kRowBytes;   // rows of one load
    const bool whole = step.k_left >= kBK;
    const char* base = step.base + (kPair && ((i * NW + wave) * kRows & 32) ? step.to_pair : 0);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, kRange, 4 << 15);
    uint32_t v = voff[i];
    if (!whole) v = k_of(i) < step.k_left ? v : 0x80000000u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(lds + (i * NW + wave) * 1024),
                                             16, v, 0, 0, 0);
  }
};

// Reads the operand fragments of 16 rows of m (or n) from a staged step: lane
// l gets row l % 16 and the eight k from 8 (l / 16) on.
template <typename T, int R, Along AL>
struct Reader {
  typedef typename Frag<T>::v8 v8;
  uint32_t off;   // kAlongK: of the lane's piece of row 0; kAlongMN: of its k row and quad
  uint32_t flip;  // kAlongMN: the XOR on its 32-byte units
  int unit;       // kAlongMN: the wave's first unit

  // first: the wave's first row within the tile, a multiple of 16
  __device__ __forceinline__ void init(int first, int lane) {
    const int g = lane >> 4, s = lane & 15;
    typedef Stage<R, 1, AL> S;
    if constexpr (AL == kAlongK) {
      off = (first + s) * (kBK * 2) + ((g ^ S::swz_k(s)) << 4);
    } else {
      const int j = s >> 2, q = s & 3, k = 8 * g + j;
      off = k * (R * 2) + q * 8;
      flip = S::swz(k) << 5;
      unit = first / 16;
    }
  }
  // Called once a step: the fragments' addresses are formed again from off and
  // flip at each read (one instruction), which takes the place of a register
  // each for the whole loop.
  __device__ __forceinline__ void fresh() {
    if constexpr (AL == kAlongMN) asm volatile("" : "+v"(flip));
  }
  __device__ __forceinline__ v8 get(const char* lds, int t) const {
    if constexpr (AL == kAlongK) {
      return *reinterpret_cast<const v8*>(lds + (off + t * 16 * (kBK * 2)));
    } else {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      typedef __attribute__((address_space(3))) s4* p4;
      // the transposing load takes four k rows from 16 lanes, each four
      // neighbouring columns of one, and gives lane s column s of all four
      const char* p = lds + ((((uint32_t)(unit + t) << 5) ^ flip) + off);
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(p + 4 * (R * 2)));
      const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(v8, v);
    }
  }
};

// Tile of WM x WN waves, each TM x TN products of 16 x 16.
template <int WM_, int WN_, int TM_, int TN_>
struct TileCfg {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_;
  static constexpr int NW = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16, kThreads = NW * 64;
};

// One staged step of both operands. The steps in flight are LDS arrays of
// their own, so that the compiler can tell the one being read from those being
// loaded and does not wait for all of them.
template <typename C>
struct LdsStep {
  char a[C::BM * kBK * 2];
  char b[C::BN * kBK * 2];
};
#define NAJU_GEMM_LDS(C)                                                        \
  __shared__ __attribute__((aligned(1024))) LdsStep<C> s_step0, s_step1, s_step2, s_step3; \
  LdsStep<C>* const s_steps[4] = {&s_step0, &s_step1, &s_step2, &s_step3}

// The products of one tile after another, by one workgroup. For each tile:
//   init(...)     the operands' strides and row maps (Stage::init);
//   start(...)    the loads of the first two steps; the LDS must be free;
//   run(...)      acc = the products of all steps; leaves the LDS free.
// start() of the next tile may come before the epilogue of this one, whose
// stores then run beside those loads. a_at(step) / b_at(step) give a step's
// base address and how many of its k exist; steps past the end count as zeros,
// so that the loop has no branches.
template <typename T, typename C, Along AA, Along AB, bool kPairB = false>
struct TilePipe {
  typedef typename Frag<T>::v8 v8;
  typedef Stage<C::BM, C::NW, AA> SA;
  typedef Stage<C::BN, C::NW, AB> SB;
  static constexpr int kPer = SA::kLoads + SB::kLoads;  // loads of one step, per wave
  SA sa;
  SB sb;
  int lane, wave;

  template <typename MapA, typename MapB>
  __device__ __forceinline__ void init(uint32_t lda, uint32_t ldb, MapA map_a, MapB map_b) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    sa.init(wave, lane, lda, map_a);
    sb.init(wave, lane, ldb, map_b);
  }

  template <typename AtA, typename AtB>
  __device__ __forceinline__ void issue(int s, int steps, AtA a_at, AtB b_at, LdsStep<C>* l) const {
    Step a = a_at(s), b = b_at(s);
    if (s >= steps) a.k_left = b.k_left = 0;
    sa.template load<false>(a, wave, l->a);
    sb.template load<kPairB>(b, wave, l->b);
  }

  template <typename AtA, typename AtB>
  __device__ __forceinline__ void start(LdsStep<C>* const (&lds)[4], int steps, AtA a_at, AtB b_at) const {
    issue(0, steps, a_at, b_at, lds[0]);
    issue(1, steps, a_at, b_at, lds[1]);
  }

  // While step s is multiplied from registers, step s + 1 is read into them
  // behind the products that used them last, and steps s + 2 and s + 3 are on
  // their way. arrive() waits until step s + 1 is in LDS (all loads but those
  // of the step after it); its barrier also has every wave past the products
  // of step s - 1, and so past the reads of it, whose LDS step s + 3 takes.
  static __device__ __forceinline__ void arrive() {
    __builtin_amdgcn_s_waitcnt(0x0f70 | (kPer & 15) | ((kPer >> 4) << 14));
    __builtin_amdgcn_s_barrier();
  }

  template <typename AtA, typename AtB>
  __device__ __forceinline__ void run(acc_t (&acc)[C::TM][C::TN], LdsStep<C>* const (&lds)[4], int steps, AtA a_at,
                                      AtB b_at) const {
    Reader<T, C::BM, AA> ra;
    Reader<T, C::BN, AB> rb;
    ra.init(wave / C::WN * C::TM * 16, lane);
    rb.init(wave % C::WN * C::TN * 16, lane);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) acc[i][j] = acc_t{0.f, 0.f, 0.f, 0.f};
    v8 fa[C::TM], fb[2][C::TN];
    arrive();
    issue(2, steps, a_at, b_at, lds[2]);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) fb[0][j] = rb.get(lds[0]->b, j);
#pragma unroll
    for (int i = 0; i < C::TM; ++i) fa[i] = ra.get(lds[0]->a, i);
    // the reads and the loads are spread over the groups of products, whose
    // time hides their addresses (all of them at the head of the step: 1265,
    // 1265 and 1225 TFLOP/s in the three layouts against 1290)
    constexpr int kFirst = 2, kPerGroup = (kPer + C::TM - kFirst - 1) / (C::TM - kFirst);
    static_assert(2 * C::TM >= C::TN, "two n fragments a group");
    // (whole fours of steps: an exit after two gained 3% where 25 steps became 26
    // in place of 28, and cost 4% everywhere in the other two layouts)
    for (int s = 0; s < steps; s += 4) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const LdsStep<C>* nxt = lds[(q + 1) & 3];
        LdsStep<C>* far = lds[(q + 3) & 3];
        arrive();
        ra.fresh();
        rb.fresh();
        Step at = a_at(s + q + 3), bt = b_at(s + q + 3);
        if (s + q + 3 >= steps) at.k_left = bt.k_left = 0;
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
#pragma unroll
          for (int j = 0; j < C::TN; ++j) acc[i][j] = Frag<T>::mma(fb[q & 1][j], fa[i], acc[i][j]);
          fa[i] = ra.get(nxt->a, i);
#pragma unroll
          for (int j = 2 * i; j < 2 * i + 2 && j < C::TN; ++j) fb[(q + 1) & 1][j] = rb.get(nxt->b, j);
#pragma unroll
          for (int u = 0; u < kPerGroup; ++u) {
            const int z = (i - kFirst) * kPerGroup + u;
            if (i >= kFirst && z < SA::kLoads) sa.template load_one<false>(at, z, wave, far->a);
            if (i >= kFirst && z >= SA::kLoads && z < kPer)
              sb.template load_one<kPairB>(bt, z - SA::kLoads, wave, far->b);
          }
          // keeps each read and load behind the products before it: the order
          // above holds two steps' fragments in the registers of one and a half
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    // the loads past the end too are in LDS before it is used for anything else
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
  }
};

// LDS rows of a kAlongK n operand in an order that gives lane l, in products 2 q
// and 2 q + 1 of its wave, the eight neighbouring columns 32 q + 8 (l / 16) ...
// + 7 (32-row groups of the tile are permuted within themselves): the epilogue
// stores 16 bytes a lane and 64 a row at once. 16384 x 12544 x 768 with its
// result stored: 447 us with rows in their own order, 394 so.
__device__ __forceinline__ int wide_row(int r) { return (r & ~31) + ((r >> 2) & 3) * 8 + ((r >> 4) & 1) * 4 + (r & 3); }

// Tile (bm, bn) of an nm x nn grid for number `id`. Workgroups, and the tiles
// that one takes in turn, go round the eight XCDs; each XCD takes one contiguous run of tiles, walked in
// groups of eight rows of tiles so that the tiles in flight on an XCD share
// their operands in its L2.
__device__ __forceinline__ void tile_of(int id, int nm, int nn, int& bm, int& bn) {
  const int total = nm * nn, x = id & 7, per = total >> 3, rem = total & 7;
  const int t = x * per + (x < rem ? x : rem) + (id >> 3);
  constexpr int G = 8;
  const int group = t / (G * nn), first = group * G;
  const int g = nm - first < G ? nm - first : G;
  const int in = t - group * G * nn;
  // uniform by construction; the divisions above leave it in vector registers
  bm = __builtin_amdgcn_readfirstlane(first + in % g);
  bn = __builtin_amdgcn_readfirstlane(in / g);
}

}  // namespace
}  // namespace naju_detail

#endif  // NAJU_GEMM_TILE_H
