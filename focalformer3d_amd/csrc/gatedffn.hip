// Gated projection of a feed-forward block, forward and backward, in fp32, bf16 and fp16:
//   h = act(g) * u,   [g | u] = x [Wg ; Wu]^T + [bg | bu]           x (M, C), weight (2 F, C), h (M, F)
// and, given dh:  dg = dh u act'(g),  du = dh act(g),  [dg | du] =: d (M, 2 F),
//   dx = d W,   dW = d^T x,   db = column sums of d.
// All four are matrix products on one tiled kernel with different operand orders and epilogues:
//   gated      both projections in one block: a wave owns the same 32 columns of g and of u, so the activation and the product
//              happen on its accumulators and g, u never reach memory
//   gated_bwd  the same products again with dh in the epilogue -> d (rounded to the type once, as the operand of the two products
//              below has to be: dx and dW are off by 1.41 times the error of a single rounding) and the column sums of the unrounded
//              d.  g and u are recomputed instead of saved: 2 M C F more multiply-adds, against 2 M F values written and read again
//              and against rounding them, which alone would make that 1.7 times.  In fp16 d is scaled first (RANGED below)
//   plain      dx and, with its row sum cut into slices that a second kernel adds in order, dW: results do not depend on timing
// A block computes C^T tiles: the n side (features of W, columns of the output) is the row operand, so a lane holds 4 consecutive
// columns of one output row and stores them together.
// Measured on one MI355X (a large library product: 1309 TFLOP/s in bf16, 154 in fp32): 16384 x 1024 -> 2736 in bf16, 184 GFLOP each: forward
// 194 .. 214 us, d 270, dx 181, dW 287 + 10 (the matrix unit is the bound; d adds reading dh and writing d, dW's 88 tiles in two slices fill
// 69 % of the chip); 2880 x 256 -> 1024 in fp32, 3 GFLOP each: 31, 39, 33, 35 us and 10 for the sums of slices (bound by splitting operands
// and by latency); 4 x 1024 -> 2736 in bf16: 8 us, the weight at 1.4 TB/s.
#include <type_traits>

#include "ff3d_mma.h"

namespace {

using namespace mma;

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2, ACT_SIGMOID = 3 };
enum { EPI_GATED = 0, EPI_GATED_BWD = 1, EPI_PLAIN = 2, EPI_PARTIAL = 3 };

struct GemmArgs {
  const char *a, *b;            // m side and n side
  long long a_bytes, b_bytes;   // sizes of both operands in memory
  long long lda, ldb, ldo;      // elements
  void* out;                    // T, or fp32 slices (EPI_PARTIAL)
  const void *bias, *dh;        // EPI_GATED*: (2 F) or NULL; (M, F)
  float* colsum;                // EPI_GATED_BWD: (m blocks, 2 F) sums of d, or NULL
  long long lddh;
  int M, N, K;                  // output rows and columns (F for EPI_GATED*), length of the sums
  int acols, bcols;             // column tiles: width of the operand, padded to whole granules
  int F, act, mt, nt, slices, kslice;
  int vec_out, vec_out2, vec_dh;     // 16-byte accesses of rows of out, of its second half (EPI_GATED_BWD) and of dh are aligned
  int out_pad;                  // EPI_GATED_BWD: zero columns behind the 2 F
  const float4* range;          // fp16 gradients: what d's scale follows from (Range), nrange of them
  int nrange;
};

// fp16 holds 2^-24 .. 2^16, and a gradient's terms need not lie there where its sums do: dh u act' overflows behind a scaled loss, or loses
// its digits below 2^-14 (dh of 1e-6 over 4096 rows: dW off by 62 times the error of one rounding).  d is therefore stored times a power of
// two, the largest with |d| < 2^15 for certain, and dx, dW and their slices are multiplied back in fp32.  The certainty is
//   |d| <= 1.14 (max_m max|dh_m| |x_m|  max_n |w_n| + max|dh| (max|b| + 1)),       |act'| <= 1.14, |act(g)| <= |g| or 1
// over finite values (one that is not gives a row that is not, whatever the scale), a few binades above the largest d of ordinary data: what is
// lost of d lies 2^-29 and more below the bound.  One scale serves the whole matrix, since dx sums over its columns and dW over its rows.
// It costs one reading of dh, x and W:
// 16384 x 1024 -> 2736 in 34 us (134 MB, 4.0 TB/s; forward and backward 915 instead of 866), 2880 x 256 -> 1024 in 6 us.
template <typename T>
constexpr bool RANGED = sizeof(T) == 2 && !std::is_same_v<T, __bf16>;
constexpr int RANGE_BLOCKS = 256, RANGE_THREADS = 1024;

__device__ __forceinline__ float max_wave(float v) {
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) v = fmaxf(v, __shfl_xor(v, x));
  return v;
}
// e of the scale 2^e, the same in every wave that asks
__device__ __forceinline__ int range_exp(const GemmArgs& p, int lane) {
  float4 m = {0.f, 0.f, 0.f, 0.f};
  for (int i = lane; i < p.nrange; i += 64) {
    const float4 r = p.range[i];
    m.x = fmaxf(m.x, r.x), m.y = fmaxf(m.y, r.y), m.z = fmaxf(m.z, r.z), m.w = fmaxf(m.w, r.w);
  }
  const float bound = 1.14f * (max_wave(m.x) * sqrtf(max_wave(m.z)) + max_wave(m.y) * (max_wave(m.w) + 1.f));
  const int ex = (int)(__float_as_uint(bound) >> 23) - 127;
  return __builtin_amdgcn_readfirstlane(bound > 0.f ? 14 - ex : 0);
}

// exp for the type: fp32 outputs take the full-precision function, 16-bit ones the hardware's exp2 of the rounded product
template <typename T>
__device__ __forceinline__ float exp_t(float x) {
  if constexpr (sizeof(T) == 4) return expf(x);
  else return __expf(x);
}

template <typename T>
__device__ __forceinline__ float sigmoid_t(float x) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-x));
  else return __builtin_amdgcn_rcpf(1.f + __expf(-x));         // 1 ulp of fp32, far below the output's rounding
}

template <typename T, int ACT>
__device__ __forceinline__ float act_f(float g) {
  if constexpr (ACT == ACT_RELU) return g < 0.f ? 0.f : g;               // a NaN stays one
  if constexpr (ACT == ACT_GELU) return g * (0.5f * (1.f + erff(g * 0.70710678118654752f)));
  const float s = sigmoid_t<T>(g);
  return ACT == ACT_SIGMOID ? s : g * s;
}
template <typename T, int ACT>
__device__ __forceinline__ void act_both(float g, float& a, float& da) {
  if constexpr (ACT == ACT_RELU) {
    a = g < 0.f ? 0.f : g, da = g > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf, da = cdf + g * exp_t<T>(-0.5f * g * g) * 0.39894228040143268f;
  } else {
    const float s = sigmoid_t<T>(g);
    if constexpr (ACT == ACT_SIGMOID) a = s, da = s * (1.f - s);
    else a = g * s, da = s * (1.f + g * (1.f - s));
  }
}

template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>{});
  else if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>{});
  else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
  else f(std::integral_constant<int, ACT_SIGMOID>{});
}

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v, int left, bool vec) {
  if (vec && left >= 4) {
    Four<T> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = from_f<T>(v[i]);
    *(Four<T>*)p = f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* v, int left, bool vec) {
  if (vec && left >= 4) {
    const Four<T> f = *(const Four<T>*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f(f.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? to_f(p[i]) : 0.f;
  }
}

// The loop over the long sum.  Blocks of 8 waves (256 x 256): steps of 64 bytes of k in a ring of four; the two waves of a SIMD work
// half a step apart, one reading its operands and asking for the step after next but one while the other multiplies, so the matrix
// unit of the SIMD is fed without a pause (dx of 16384 x 1024 over 5472 in bf16: 182 us, against 217 with two steps of 128 bytes that
// all waves read, multiply and wait for together).  Blocks of 4 waves: two or more share a CU and fill each other's waits; two steps
// of 128 bytes (128 x 128, the same product: 221 us, 250 with the ring).
constexpr int step_bytes_of(int waves) { return waves == 8 ? 64 : 128; }
constexpr int stages_of(int waves) { return waves == 8 ? 4 : 2; }

// One operand of a block: ROWS rows (or columns) of it, BK of k per step, DMA-ed into LDS.
// ROW: k is contiguous in memory (row tile), else the rows are (column tile).  DUAL: rows come in blocks of 32 alternating between
// the gate and the value half of the weight.
template <typename T, bool ROW, bool DUAL, int ROWS, int NT>
struct Operand {
  static constexpr int STEP = step_bytes_of(NT / 64), P = Type<T>::PER16, BK = STEP / (int)sizeof(T), GK = STEP / 16, N = ROWS * GK / NT;
  static_assert(ROWS * GK % NT == 0, "whole granules per thread");
  const char *base, *end;
  long long step_bytes;
  unsigned off[N];
  int kk[N];                     // k of the granule inside a step

  __device__ __forceinline__ void init(const char* p, long long bytes, long long ld, int row0, int nrows, int half_rows, long long k0, int tid) {
    end = p + bytes;
    if constexpr (ROW) {
      base = p + (DUAL ? 0 : (long long)row0 * ld * sizeof(T)) + k0 * (long long)sizeof(T);
      step_bytes = STEP;
    } else {
      base = p + k0 * ld * (long long)sizeof(T) + (long long)row0 * sizeof(T);
      step_bytes = (long long)BK * ld * sizeof(T);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * NT + tid;
      if constexpr (ROW) {
        const int r = at / GK, g = place<GK>(r, at % GK);
        int row = r;
        bool in = row0 + r < nrows;
        if constexpr (DUAL) {
          const int f = row0 + (r >> 6) * 32 + (r & 31);
          in = f < nrows;
          row = f + ((r >> 5) & 1) * half_rows;
        }
        kk[i] = g * P;
        off[i] = in ? (unsigned)row * (unsigned)(ld * sizeof(T)) + g * 16u : OUT;
      } else {
        constexpr int GR = ROWS / P;
        const int k = at / GR, g = place<GR>(k, at % GR);
        kk[i] = k;
        off[i] = row0 + g * P < nrows ? (unsigned)k * (unsigned)(ld * sizeof(T)) + g * 16u : OUT;
      }
    }
  }
  // the step whose k runs over `left` more elements, into `lds`
  __device__ __forceinline__ void stage(char* lds, int wave, int left) {
    const rsrc_t r = make_rsrc(base, end - base);
#pragma unroll
    for (int i = 0; i < N; ++i) load_lds16(r, lds + (i * NT + wave * 64) * 16, kk[i] < left ? off[i] : OUT);
    base += step_bytes;
  }
};

template <typename T, bool AROW, bool BROW, int WM, int WN, int TM, int TN, int EPI>
__global__ __launch_bounds__(WM* WN * 64) void gemm_kernel(GemmArgs p) {
  constexpr bool DUAL = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
  constexpr int NT = WM * WN * 64, BM = WM * TM * 32, BN = WN * TN * 32, BNO = DUAL ? BN / 2 : BN;
  constexpr int STEP = step_bytes_of(WM * WN), STAGES = stages_of(WM * WN), BK = STEP / (int)sizeof(T), STEPS = BK / 16, P = Type<T>::PER16, GK = STEP / 16;
  constexpr int ABYTES = BM * STEP, STAGE = (BM + BN) * STEP;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
  const int wm = wave % WM, wn = wave / WM;
  const int tiles = p.mt * p.nt;
  const int bid = (int)ff3d_xcd_remap(blockIdx.x, gridDim.x);
  const int slice = bid / tiles, tile = bid % tiles;
  // tiles in bands of 8 m blocks: the blocks that run together on an XCD share both operands' rows in its L2
  const int band = tile / (8 * p.nt), in_band = tile % (8 * p.nt), bm_n = min(8, p.mt - band * 8);
  const int mb = band * 8 + in_band % bm_n, nb = in_band / bm_n;
  const int m0 = mb * BM, n0 = nb * BNO;
  const int k0 = slice * p.kslice, kn = min(p.K - k0, p.kslice);

  Operand<T, AROW, false, BM, NT> A;
  Operand<T, BROW, DUAL, BN, NT> B;
  A.init(p.a, p.a_bytes, p.lda, m0, AROW ? p.M : p.acols, 0, k0, tid);
  B.init(p.b, p.b_bytes, p.ldb, n0, BROW ? p.N : p.bcols, p.F, k0, tid);

  f32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = (f32x16)(0.f);

  const int nk = (kn + BK - 1) / BK;
  auto stage = [&](int t) {
    char* to = lds + (t % STAGES) * STAGE;
    A.stage(to, wave, kn - t * BK);
    B.stage(to + ABYTES, wave, kn - t * BK);
  };
  vec8<T> fa[2][TM], fb[2][TN];
  auto read = [&](const char* cur, int s) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      if constexpr (AROW) fa[s & 1][j] = row_frag<T, GK>(cur, (wm * TM + j) * 32 + (lane & 31), 16 * s, half);
      else fa[s & 1][j] = col_frag<T, BM / P>(cur, 16 * s, (wm * TM + j) * 32, lane);
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      if constexpr (BROW) fb[s & 1][i] = row_frag<T, GK>(cur + ABYTES, (wn * TN + i) * 32 + (lane & 31), 16 * s, half);
      else fb[s & 1][i] = col_frag<T, BN / P>(cur + ABYTES, 16 * s, (wn * TN + i) * 32, lane);
    }
  };
  auto multiply = [&](int s) {
    Op<T> oa[TM], ob[TN];
#pragma unroll
    for (int j = 0; j < TM; ++j) oa[j] = op<T>(fa[s & 1][j]);
#pragma unroll
    for (int i = 0; i < TN; ++i) ob[i] = op<T>(fb[s & 1][i]);
    auto all = [&](auto part) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = mfma_part<decltype(part)::value>(ob[i], oa[j], acc[i][j]);
    };
    all(std::integral_constant<int, 0>{});
    if constexpr (PARTS<T> == 6) {
      all(std::integral_constant<int, 1>{}), all(std::integral_constant<int, 2>{}), all(std::integral_constant<int, 3>{});
      all(std::integral_constant<int, 4>{}), all(std::integral_constant<int, 5>{});
    }
  };
  if constexpr (WM * WN == 8) {
    // Barriers are numbered; the late half of the waves meets one before it starts.  Early waves read step t between barriers 2 t and
    // 2 t + 1 and multiply it until 2 t + 2, late ones are one barrier behind.  At the end of its reading of step t a wave has waited
    // for its own loads of step t + 1: the early waves' first look at that step comes behind two barriers, the late ones' behind
    // one.  The load of step t + 3 takes the place of step t - 1, which the late waves have read (lgkmcnt 0) before barrier 2 t.
    static_assert(STEPS == 2 && STAGES == 4, "the schedule above");
    constexpr int LOADS = Operand<T, AROW, false, BM, NT>::N + Operand<T, BROW, DUAL, BN, NT>::N;     // of a wave per step
#pragma unroll
    for (int t = 0; t < 3; ++t)
      if (t < nk) stage(t);
    if (nk > 2) wait_barrier<2 * LOADS>();
    else wait_barrier<0>();
    const bool late = wave >= 4;
    if (late) asm volatile("s_barrier" ::: "memory");
    for (int t = 0; t < nk; ++t) {
      const char* cur = lds + (t % STAGES) * STAGE;
      read(cur, 0);
      read(cur, 1);
      if (t + 3 < nk) {
        stage(t + 3);
        wait_barrier<2 * LOADS>();
      } else if (t + 2 < nk) {
        wait_barrier<LOADS>();
      } else {
        wait_barrier<0>();
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      multiply(0);
      multiply(1);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_barrier" ::: "memory");
    }
    if (!late) asm volatile("s_barrier" ::: "memory");
  } else {
    stage(0);
    for (int t = 0; t < nk; ++t) {
      const char* cur = lds + (t % STAGES) * STAGE;
      wait_barrier<0>();           // step t has arrived, and nobody reads the other half any more
      if (t + 1 < nk) stage(t + 1);
      read(cur, 0);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {      // operands of the next 16 k are read while the matrix unit works on these
        if (s + 1 < STEPS) read(cur, s + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(s);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
  }
  // Nobody reads operands any more: LDS now takes the output tile, so that it leaves (and dh arrives) in whole rows.  A lane holds 4
  // columns of a row; granule and half of the granule are swizzled by the row.

  constexpr int GO = BNO * (int)sizeof(T) / 16;      // granules of an output row
  auto out_at = [](int r, int n) {                   // byte of columns n .. n + 3 (n a multiple of 4) of row r in the tile
    if constexpr (sizeof(T) == 4) return (r * GO + place<GO>(r, n / 4)) * 16;
    else return (r * GO + place<GO>(r, n / 8)) * 16 + (((n >> 2) ^ (r >> 4)) & 1) * 8;
  };
  // rows of the tile at `tile` to out + row * ldo + n0 (or fp16 / bf16 halves of a granule put back in order first)
  auto store_tile = [&](const char* tile, T* out, long long ldo, int n_end, bool vec) {
    constexpr int ITEMS = BM * GO / NT;
#pragma unroll 4
    for (int it = 0; it < ITEMS; ++it) {
      const int at = it * NT + tid, r = at / GO, g = at % GO, m = m0 + r, n = n0 + g * P, left = n_end - n;
      if (m >= p.M || left <= 0) continue;
      u32x4 v = *(const u32x4*)(tile + (r * GO + place<GO>(r, g)) * 16);
      if constexpr (sizeof(T) == 2)
        if ((r >> 4) & 1) v = (u32x4){v[2], v[3], v[0], v[1]};
      T* to = out + (long long)m * ldo + n;
      if (vec && left >= P) {
        *(u32x4*)to = v;
      } else {
        const T* e = (const T*)&v;
#pragma unroll
        for (int i = 0; i < P; ++i)
          if (i < left) to[i] = e[i];
      }
    }
  };

  if constexpr (DUAL) {
    constexpr int TILE = BM * GO * 16;
    static_assert((EPI == EPI_GATED ? 1 : 2) * TILE <= STAGES * STAGE, "the tiles fit where the operands were");
    const T* bias = (const T*)p.bias;
    float* sums = (float*)lds;     // EPI_GATED_BWD: column sums of the waves, [WM][2][BNO], once the tiles have left
    if constexpr (EPI == EPI_GATED_BWD) {
      constexpr int ITEMS = BM * GO / NT;
#pragma unroll 4
      for (int it = 0; it < ITEMS; ++it) {           // dh, in the layout of the output tile
        const int at = it * NT + tid, r = at / GO, g = at % GO, m = m0 + r, n = n0 + g * P, left = p.N - n;
        u32x4 v = (u32x4)(0u);
        if (m < p.M && left > 0) {
          const T* from = (const T*)p.dh + (long long)m * p.lddh + n;
          if (p.vec_dh && left >= P) {
            v = *(const u32x4*)from;
          } else {
            T* e = (T*)&v;
#pragma unroll
            for (int i = 0; i < P; ++i)
              if (i < left) e[i] = from[i];
          }
        }
        if constexpr (sizeof(T) == 2)
          if ((r >> 4) & 1) v = (u32x4){v[2], v[3], v[0], v[1]};
        *(u32x4*)(lds + (r * GO + place<GO>(r, g)) * 16) = v;
      }
      __syncthreads();
    }
    float sg[TN / 2][4][4] = {}, su[TN / 2][4][4] = {}, scale = 1.f;
    if constexpr (RANGED<T> && EPI == EPI_GATED_BWD) scale = ff3d_pow2(range_exp(p, lane));
    with_act(p.act, [&](auto act) {                  // outside the loops: the elements' chains run beside each other
    constexpr int ACT = decltype(act)::value;
#pragma unroll
    for (int pr = 0; pr < TN / 2; ++pr)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int nl = (wn * (TN / 2) + pr) * 32 + 8 * q + 4 * half, left = p.N - n0 - nl;
        float bg[4] = {}, bu[4] = {};
        if (bias && left > 0) {
          load4(bias + n0 + nl, bg, left, false);
          load4(bias + p.F + n0 + nl, bu, left, false);
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int r = (wm * TM + j) * 32 + (lane & 31);
          char* at = lds + out_at(r, nl);
          float g[4], u[4], o[4], o2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = acc[2 * pr][j][4 * q + i] + bg[i], u[i] = acc[2 * pr + 1][j][4 * q + i] + bu[i];
          if constexpr (EPI == EPI_GATED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = act_f<T, ACT>(g[i]) * u[i];
          } else {
            float d[4];
            load4((const T*)at, d, 4, true);         // zeros outside the matrix
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float a, da;
              act_both<T, ACT>(g[i], a, da);
              o[i] = d[i] * u[i] * da, o2[i] = d[i] * a;
              sg[pr][q][i] += o[i], su[pr][q][i] += o2[i];
              if constexpr (RANGED<T>) o[i] *= scale, o2[i] *= scale;
            }
            store4((T*)(at + TILE), o2, 4, true);
          }
          store4((T*)at, o, 4, true);                // a lane's own place, also where it held dh
        }
      }
    });
    __syncthreads();
    store_tile(lds, (T*)p.out, p.ldo, p.N, p.vec_out);
    if constexpr (EPI == EPI_GATED_BWD) {
      store_tile(lds + TILE, (T*)p.out + p.F, p.ldo, p.N, p.vec_out2);
      if (p.out_pad && n0 + BNO >= p.N)              // the operand of the next products is whole granules wide: zeros behind the 2 F
        for (int r = tid; r < BM; r += NT)
          if (m0 + r < p.M)
            for (int i = 0; i < p.out_pad; ++i) ((T*)p.out)[(long long)(m0 + r) * p.ldo + 2 * p.F + i] = from_f<T>(0.f);
      if (p.colsum) {
        __syncthreads();
#pragma unroll
        for (int pr = 0; pr < TN / 2; ++pr)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int nl = (wn * (TN / 2) + pr) * 32 + 8 * q + 4 * half + i;
#pragma unroll
              for (int x = 1; x < 32; x <<= 1) sg[pr][q][i] += __shfl_xor(sg[pr][q][i], x), su[pr][q][i] += __shfl_xor(su[pr][q][i], x);
              if ((lane & 31) == 0) sums[(wm * 2 + 0) * BNO + nl] = sg[pr][q][i], sums[(wm * 2 + 1) * BNO + nl] = su[pr][q][i];
            }
        __syncthreads();
        for (int i = tid; i < 2 * BNO; i += NT) {
          const int part = i / BNO, nl = i % BNO;
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < WM; ++w) s += sums[(w * 2 + part) * BNO + nl];
          if (n0 + nl < p.N) p.colsum[(long long)mb * 2 * p.F + part * p.F + n0 + nl] = s;
        }
      }
    }
  } else if constexpr (EPI == EPI_PLAIN) {
    static_assert(BM * GO * 16 <= STAGES * STAGE, "the tile fits where the operands were");
    float undo = 1.f;
    if constexpr (RANGED<T>) undo = ff3d_pow2(-range_exp(p, lane));
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = RANGED<T> ? acc[i][j][4 * q + e] * undo : acc[i][j][4 * q + e];
          store4((T*)(lds + out_at((wm * TM + j) * 32 + (lane & 31), (wn * TN + i) * 32 + 8 * q + 4 * half)), o, 4, true);
        }
    __syncthreads();
    store_tile(lds, (T*)p.out, p.ldo, p.N, p.vec_out);
  } else {
    float undo = 1.f;
    if constexpr (RANGED<T>) undo = ff3d_pow2(-range_exp(p, lane));
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + (wn * TN + i) * 32 + 8 * q + 4 * half, left = p.N - n;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int m = m0 + (wm * TM + j) * 32 + (lane & 31);
          if (m < p.M && left > 0) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = RANGED<T> ? acc[i][j][4 * q + e] * undo : acc[i][j][4 * q + e];
            store4((float*)p.out + ((long long)slice * p.M + m) * p.ldo + n, o, left, p.vec_out);
          }
        }
      }
  }
}

// Few rows: a block computes 32 columns of h for 32 rows, its waves taking every NW-th piece of 128 bytes of k.  Bound by reading the
// weight once: operands go straight from memory to registers, a lane reading 64 contiguous bytes (its half of the piece: the order of
// k is the same for both operands, which is all a product needs), and nothing is waited for but the data itself.
template <typename T, int NW>
__global__ __launch_bounds__(NW * 64) void gated_rows_kernel(GemmArgs p) {
  constexpr int STEPS = 8 / (int)sizeof(T), PIECE = 128 / (int)sizeof(T), P = Type<T>::PER16;
  __shared__ float sums[NW][2][16][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const int nb = blockIdx.x % p.nt, n0 = nb * 32, m0 = blockIdx.x / p.nt * 32;
  const int n = n0 + (lane & 31), m = m0 + (lane & 31);
  const char* pg = p.b + (long long)min(n, p.N - 1) * p.ldb * (long long)sizeof(T) + half * 64;
  const char* pu = pg + (long long)p.F * p.ldb * (long long)sizeof(T);
  const char* px = p.a + (long long)min(m, p.M - 1) * p.lda * (long long)sizeof(T) + half * 64;
  f32x16 acc[2] = {(f32x16)(0.f), (f32x16)(0.f)};
  const int pieces = (p.K + PIECE - 1) / PIECE;
#pragma unroll 2
  for (int c = wave; c < pieces; c += NW) {
    u32x4 g[4], u[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = c * PIECE + half * (PIECE / 2) + i * P < p.K;
      const long long at = (long long)c * 128 + i * 16;
      g[i] = in ? *(const u32x4*)(pg + at) : (u32x4)(0u);
      u[i] = in ? *(const u32x4*)(pu + at) : (u32x4)(0u);
      x[i] = in ? *(const u32x4*)(px + at) : (u32x4)(0u);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const Op<T> ox = op<T>(((const vec8<T>*)x)[s]);
      acc[0] = mfma_step<T>(op<T>(((const vec8<T>*)g)[s]), ox, acc[0]);
      acc[1] = mfma_step<T>(op<T>(((const vec8<T>*)u)[s]), ox, acc[1]);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[wave][t][e][lane] = acc[t][e];
  __syncthreads();
  const T* bias = (const T*)p.bias;
  with_act(p.act, [&](auto act) {
  constexpr int ACT = decltype(act)::value;
  for (int it = threadIdx.x; it < 1024; it += NW * 64) {         // (row, column) pairs, columns running fastest
    const int nl = it & 31, ml = it >> 5, e = 4 * (nl >> 3) + (nl & 3), at = ml + 32 * ((nl >> 2) & 1);
    if (n0 + nl >= p.N || m0 + ml >= p.M) continue;
    float g = bias ? to_f(bias[n0 + nl]) : 0.f, u = bias ? to_f(bias[p.F + n0 + nl]) : 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) g += sums[w][0][e][at], u += sums[w][1][e][at];
    ((T*)p.out)[(long long)(m0 + ml) * p.ldo + n0 + nl] = from_f<T>(act_f<T, ACT>(g) * u);
  }
  });
}

// Range, one per block: max_m max|dh_m| |x_m|, max|dh|, max_n |w_n|^2, max|b|, all over finite values.  A wave takes a row of dh and of x, or
// one of the weight, at a time; rows of x and of the weight are whole aligned granules (K elements, zeros behind their own).
template <typename T>
__global__ __launch_bounds__(RANGE_THREADS) void range_kernel(GemmArgs p, float4* range) {
  constexpr int P = Type<T>::PER16;
  __shared__ float4 found[RANGE_THREADS / 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float4 m = {0.f, 0.f, 0.f, 0.f};
  auto finite = [](T v) {
    const float a = fabsf(to_f(v));
    return a < INFINITY ? a : 0.f;                   // a NaN compares false
  };
  auto largest = [&](const T* row, int n, bool vec) {
    float top = 0.f;
    int c = lane * P;
    if (vec) {
#pragma unroll 4
      for (; c + P <= n; c += 64 * P) {
        const vec8<T> v = *(const vec8<T>*)(row + c);
#pragma unroll
        for (int e = 0; e < P; ++e) top = fmaxf(top, finite(v[e]));
      }
      for (int e = c; e < min(c + P, n); ++e) top = fmaxf(top, finite(row[e]));
    } else {
#pragma unroll 4
      for (int e = lane; e < n; e += 64) top = fmaxf(top, finite(row[e]));
    }
    return max_wave(top);
  };
  auto squares = [&](const char* row) {
    float s = 0.f;
#pragma unroll 4
    for (int c = lane * P; c < p.K; c += 64 * P) {
      const vec8<T> v = *(const vec8<T>*)(row + c * (int)sizeof(T));
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float a = finite(v[e]);
        s = fmaf(a, a, s);
      }
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) s += __shfl_xor(s, x);
    return s;
  };
  const long long rows = p.M + 2ll * p.F;
  for (long long r = (long long)blockIdx.x * (RANGE_THREADS / 64) + wave; r < rows; r += (long long)gridDim.x * (RANGE_THREADS / 64)) {
    if (r < p.M) {
      const float top = largest((const T*)p.dh + r * p.lddh, p.F, p.vec_dh);
      m.x = fmaxf(m.x, top * sqrtf(squares(p.a + r * p.lda * (long long)sizeof(T)))), m.y = fmaxf(m.y, top);
    } else {
      const long long n = r - p.M;
      m.z = fmaxf(m.z, squares(p.b + n * p.ldb * (long long)sizeof(T)));
      if (p.bias) m.w = fmaxf(m.w, finite(((const T*)p.bias)[n]));
    }
  }
  if (lane == 0) found[wave] = m;                    // the same in every lane
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < RANGE_THREADS / 64; ++w) {
      const float4 o = found[w];
      m.x = fmaxf(m.x, o.x), m.y = fmaxf(m.y, o.y), m.z = fmaxf(m.z, o.z), m.w = fmaxf(m.w, o.w);
    }
    range[blockIdx.x] = m;
  }
}

// out[i] = sum of the slices part[k n + i] in order
template <typename T>
struct SumJob {
  const float* part;
  T* out;
  long long n;
  int slices, blocks, wide;       // wide: four elements per thread
};
template <typename T, int W>
__device__ __forceinline__ void sum_slices(const SumJob<T>& j, int block) {
  struct alignas(4 * W) In { float v[W]; };
  struct alignas(W * sizeof(T)) Out { T v[W]; };
  for (long long i = (long long)block * 256 + threadIdx.x; i < j.n / W; i += (long long)j.blocks * 256) {
    float s[W] = {};
#pragma unroll 8
    for (int k = 0; k < j.slices; ++k) {
      const In v = ((const In*)(j.part + k * j.n))[i];
#pragma unroll
      for (int e = 0; e < W; ++e) s[e] += v.v[e];
    }
    Out o;
#pragma unroll
    for (int e = 0; e < W; ++e) o.v[e] = from_f<T>(s[e]);
    ((Out*)j.out)[i] = o;
  }
}
// the slices of dx, of dW and the column sums of d, in one launch behind the products
template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(SumJob<T> j0, SumJob<T> j1, SumJob<T> j2) {
  int at = blockIdx.x;
  SumJob<T> j = j0;
  if (at >= j.blocks) {
    at -= j.blocks, j = j1;
    if (at >= j.blocks) at -= j.blocks, j = j2;
  }
  if (j.wide) sum_slices<T, 4>(j, at);
  else sum_slices<T, 1>(j, at);
}
template <typename T>
SumJob<T> sum_job(const float* part, T* out, int slices, long long n) {
  const int wide = n % 4 == 0 && ff3d_aligned16(out);
  const long long items = wide ? n / 4 : n, blocks = (items + 255) / 256;
  return {part, out, n, slices, (int)(blocks < 2048 ? blocks : 2048), wide};
}

// rows of `cols` elements with stride ld into rows of whole granules, zeros behind
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* src, long long ld, T* dst, int rows, int cols, int padded) {
  const long long n = (long long)rows * padded;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / padded;
    const int c = (int)(i - r * padded);
    dst[i] = c < cols ? src[r * ld + c] : from_f<T>(0.f);
  }
}

inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }
inline long long align_up(long long a, long long b) { return (a + b - 1) / b * b; }
inline int grid_for(long long n) { return (int)(n < 1024ll * 256 ? (n + 255) / 256 : 1024); }

template <typename T, bool AROW, bool BROW, int WM, int WN, int TM, int TN, int EPI>
int launch(GemmArgs a, hipStream_t st) {
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, BNO = (EPI == EPI_GATED || EPI == EPI_GATED_BWD) ? BN / 2 : BN;
  constexpr int LDS = stages_of(WM * WN) * (BM + BN) * step_bytes_of(WM * WN);
  auto k = gemm_kernel<T, AROW, BROW, WM, WN, TM, TN, EPI>;
  if (LDS > 64 * 1024) (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  a.mt = cdiv(a.M, BM), a.nt = cdiv(a.N, BNO);
  const long long blocks = (long long)a.mt * a.nt * a.slices;
  if (blocks > 0x7fffffffll) return FF3D_ERR_BAD_SHAPE;
  k<<<(unsigned)blocks, WM * WN * 64, LDS, st>>>(a);
  return ff3d_launch_status();
}

// Which tile, and into how many slices a long sum is cut: the least of an estimate in microseconds.  Blocks run in rounds that fill the
// chip's places; an element of k takes a round between `alone` (one block on a few CUs: latency) and `full` (every place taken), half by
// how many places are taken and half by how many on the fullest CU, and the first round its filling and draining, which grow with it.  Slices cost their fp32 sums, written and read at 4.5 TB/s, and a launch.
// Measured on 600 .. 16384 rows of 112 .. 1024 columns to 192 .. 2736 and both gradients: e.g. 1024 x 1024 -> 2736 forward in bf16 17 us
// in 128 x 128 tiles, 27 in 256 x 256 ones; 2880 x 256 -> 1024 8 us in 64 x 128 tiles, 13 in 256 x 256 ones; 16384 x 5472 x 1024 190 us in
// 256 x 256 tiles, 225 in 128 x 128 ones.
inline long long slice_length(long long K, int slices) { return align_up(cdiv(K, slices), 64); }

struct Tile {
  int id, bm, bn, slices;
};
template <typename T>
Tile pick(long long M, long long N, long long K, bool dual, bool cut) {
  const int half = dual ? 2 : 1;
  constexpr bool F32 = sizeof(T) == 4;
  const struct { int bm, bn, per_cu; double alone, full, fixed; } t[3] = {
      {256, 256 / half, 1, 0.0184, 0.029, 6.0},
      {128, 128 / half, 2, F32 ? 0.047 : 0.0113, F32 ? 0.075 : 0.0165, F32 ? 6.0 : 3.0},
      {64, 128 / half, 3, F32 ? 0.033 : 0.0105, F32 ? 0.073 : 0.0155, F32 ? 5.0 : 2.5}};
  Tile best = {2, t[2].bm, t[2].bn, 1};
  double least = 1e300;
  for (int i = F32 ? 1 : 0; i < 3; ++i)
    for (int s = 1; s <= (cut ? 16 : 1) && (s == 1 || K / s >= 128); ++s) {
      const long long k = s > 1 ? slice_length(K, s) : K;
      const long long blocks = (long long)cdiv(M, t[i].bm) * cdiv(N, t[i].bn) * cdiv(K, k), slots = 256ll * t[i].per_cu;
      const double part = (double)(blocks % slots) / slots, deep = t[i].per_cu > 1 ? (double)cdiv(blocks % slots, 256) / t[i].per_cu : part;
      const double rest = 0.5 * (part + deep), first = blocks < slots ? rest : 1.0;
      const double round = t[i].alone + (t[i].full - t[i].alone) * rest;
      const double cost = t[i].fixed * (1 + first) + k * ((double)(blocks / slots) * t[i].full + (rest > 0 ? round : 0)) +
                          (s > 1 ? 5 + s * (double)M * N * 8 / 4.5e6 : 0);
      if (cost < least) least = cost, best = {i, t[i].bm, t[i].bn, s};
    }
  return best;
}

template <typename T, bool AROW, bool BROW, int EPI>
int dispatch(const Tile& t, const GemmArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (t.id == 0) return launch<T, AROW, BROW, 2, 4, 4, 2, EPI>(a, st);
  if (t.id <= 1) return launch<T, AROW, BROW, 2, 2, 2, 2, EPI>(a, st);
  return launch<T, AROW, BROW, 2, 2, 1, 2, EPI>(a, st);
}

struct Plan {                    // of one call: packed operands, partial sums, and where they lie in the workspace
  int P, Cp, ldd, mblocks;
  long long x, w, d, part, part_w, colsum, range, total;
};
// bytes of the slices of a product of M x N over K (0: one piece), and their length
template <typename T>
long long slices_of(const Tile& t, long long M, long long N, long long K, int* kslice, int* slices) {
  *kslice = t.slices > 1 ? (int)slice_length(K, t.slices) : (int)K;
  *slices = cdiv(K, *kslice);
  return *slices > 1 ? *slices * M * N * 4 : 0;
}
template <typename T>
Plan plan(long long M, int C, int F, int pack, bool bwd) {
  Plan p;
  p.P = Type<T>::PER16;
  p.Cp = (int)align_up(C, p.P);
  p.ldd = (int)align_up(2ll * F, p.P);
  long long at = 0;
  auto take = [&](long long bytes) { const long long o = at; at += align_up(bytes, 256); return o; };
  p.x = (pack & 1) ? take(M * p.Cp * sizeof(T)) : 0;
  p.w = (pack & 2) ? take(2ll * F * p.Cp * sizeof(T)) : 0;
  p.mblocks = 0, p.d = p.part = p.part_w = p.colsum = p.range = 0;
  if (bwd) {
    p.d = take(M * p.ldd * sizeof(T));
    p.mblocks = cdiv(M, pick<T>(M, F, p.Cp, true, false).bm);
    p.colsum = take((long long)p.mblocks * 2 * F * 4);
    int k, n;
    const long long dx = slices_of<T>(pick<T>(M, C, 2ll * F, false, true), M, C, 2ll * F, &k, &n);
    const long long dw = slices_of<T>(pick<T>(2ll * F, C, M, false, true), 2ll * F, C, M, &k, &n);
    p.part = take(dx), p.part_w = take(dw);
    if (RANGED<T>) p.range = take(RANGE_BLOCKS * sizeof(float4));
  }
  p.total = at;
  return p;
}

template <typename T>
void pack_operands(const Plan& pl, int pack, const T*& x, long long& ldx, const T*& w, long long& ldw, long long M, int C, int F, char* ws, hipStream_t st) {
  if (pack & 1) {
    pack_kernel<T><<<grid_for(M * pl.Cp), 256, 0, st>>>(x, ldx, (T*)(ws + pl.x), (int)M, C, pl.Cp);
    x = (const T*)(ws + pl.x), ldx = pl.Cp;
  }
  if (pack & 2) {
    pack_kernel<T><<<grid_for(2ll * F * pl.Cp), 256, 0, st>>>(w, ldw, (T*)(ws + pl.w), 2 * F, C, pl.Cp);
    w = (const T*)(ws + pl.w), ldw = pl.Cp;
  }
}

template <typename T>
GemmArgs gated_args(const T* x, long long ldx, const T* w, long long ldw, const T* bias, int M, int C, int Cp, int F, int act) {
  GemmArgs a = {};
  a.a = (const char*)x, a.b = (const char*)w, a.lda = ldx, a.ldb = ldw;
  a.a_bytes = ((M - 1) * ldx + Cp) * (long long)sizeof(T), a.b_bytes = ((2ll * F - 1) * ldw + Cp) * (long long)sizeof(T);
  a.bias = bias, a.M = M, a.N = F, a.K = Cp, a.F = F, a.act = act, a.slices = 1, a.kslice = Cp;
  return a;
}

// rows of stride ld (elements) at p may be accessed 16 bytes at a time
inline bool vec_ok(const void* p, long long ld, int size) { return ld * size % 16 == 0 && ff3d_aligned16(p); }

template <typename T>
int fwd(const T* x, long long ldx, const T* w, const T* bias, T* h, int M, int C, int F, int act, int pack, char* ws, hipStream_t st) {
  const Plan pl = plan<T>(M, C, F, pack, false);
  long long ldw = C;
  pack_operands<T>(pl, pack, x, ldx, w, ldw, M, C, F, ws, st);
  GemmArgs a = gated_args<T>(x, ldx, w, ldw, bias, M, C, pl.Cp, F, act);
  a.out = h, a.ldo = F, a.vec_out = vec_ok(h, F, sizeof(T));
  const long long small = (long long)cdiv(M, 32) * cdiv(F, 32);
  // Few rows / tiles, in us.  1024 -> 2736: bf16 7.9 / 9.2 at 4 rows, 9.0 / 9.3 at 8, 9.9 / 9.3 at 12, 15.9 / 9.5 at 33, fp32 14 / 37 at 4,
  // 25 / 38 at 64, 36 / 38 at 96, 39 / 38 at 128.  256 -> 1024: bf16 4.9 / 4.9 at 8, 5.4 / 5.0 at 12, fp32 6.7 / 12.2 at 4, 10.3 / 12.7 at 96,
  // 19.5 / 13.3 at 600.  The same at 512 -> 512 and 1536 -> 4096, and in fp16.
  if (M <= (sizeof(T) == 2 ? 8 : 96)) {
    a.nt = cdiv(F, 32);
    if (pl.Cp * (int)sizeof(T) >= 2048) gated_rows_kernel<T, 8><<<(unsigned)small, 512, 0, st>>>(a);
    else gated_rows_kernel<T, 4><<<(unsigned)small, 256, 0, st>>>(a);
    return ff3d_launch_status();
  }
  return dispatch<T, true, true, EPI_GATED>(pick<T>(M, F, pl.Cp, true, false), a, st);
}

// out (a.M x a.N) = the sum over a.K, in one piece or in slices that `sum` is then to add
template <typename T, bool AROW, bool BROW>
int product(GemmArgs a, T* out, float* part, SumJob<T>& sum, hipStream_t st) {
  const Tile t = pick<T>(a.M, a.N, a.K, false, true);
  slices_of<T>(t, a.M, a.N, a.K, &a.kslice, &a.slices);
  a.ldo = a.N;
  if (a.slices == 1) {
    a.out = out, a.vec_out = vec_ok(out, a.N, sizeof(T));
    return dispatch<T, AROW, BROW, EPI_PLAIN>(t, a, st);
  }
  a.out = part, a.vec_out = a.N % 4 == 0;
  sum = sum_job<T>(part, out, a.slices, (long long)a.M * a.N);
  return dispatch<T, AROW, BROW, EPI_PARTIAL>(t, a, st);
}

template <typename T>
int bwd(const T* x, long long ldx, const T* w, const T* bias, const T* dh, long long lddh, T* dx, T* dw, T* db, int M, int C, int F, int act,
        int pack, char* ws, hipStream_t st) {
  const Plan pl = plan<T>(M, C, F, pack, true);
  long long ldw = C;
  pack_operands<T>(pl, pack, x, ldx, w, ldw, M, C, F, ws, st);
  T* d = (T*)(ws + pl.d);
  float4* range = (float4*)(ws + pl.range);
  int nrange = 0;
  {
    GemmArgs a = gated_args<T>(x, ldx, w, ldw, bias, M, C, pl.Cp, F, act);
    a.out = d, a.ldo = pl.ldd, a.dh = dh, a.lddh = lddh, a.colsum = db ? (float*)(ws + pl.colsum) : nullptr;
    a.out_pad = pl.ldd - 2 * F, a.vec_out = 1, a.vec_out2 = F * sizeof(T) % 16 == 0, a.vec_dh = vec_ok(dh, lddh, sizeof(T));
    if constexpr (RANGED<T>) {
      const int rows = cdiv(M + 2ll * F, RANGE_THREADS / 64);
      nrange = rows < RANGE_BLOCKS ? rows : RANGE_BLOCKS;
      range_kernel<T><<<nrange, RANGE_THREADS, 0, st>>>(a, range);
      a.range = range, a.nrange = nrange;
    }
    const int s = dispatch<T, true, true, EPI_GATED_BWD>(pick<T>(M, F, pl.Cp, true, false), a, st);
    if (s != FF3D_OK) return s;
  }
  const long long d_bytes = (long long)M * pl.ldd * sizeof(T);
  SumJob<T> sum_x = {}, sum_w = {}, sum_b = {};
  if (dx) {
    GemmArgs a = {};
    a.a = (const char*)d, a.lda = pl.ldd, a.a_bytes = d_bytes;
    a.b = (const char*)w, a.ldb = ldw, a.b_bytes = ((2ll * F - 1) * ldw + pl.Cp) * (long long)sizeof(T), a.bcols = pl.Cp;
    a.M = M, a.N = C, a.K = 2 * F, a.range = range, a.nrange = nrange;
    const int s = product<T, true, false>(a, dx, (float*)(ws + pl.part), sum_x, st);
    if (s != FF3D_OK) return s;
  }
  if (dw) {
    GemmArgs a = {};
    a.a = (const char*)d, a.lda = pl.ldd, a.a_bytes = d_bytes, a.acols = pl.ldd;
    a.b = (const char*)x, a.ldb = ldx, a.b_bytes = ((M - 1) * ldx + pl.Cp) * (long long)sizeof(T), a.bcols = pl.Cp;
    a.M = 2 * F, a.N = C, a.K = M, a.range = range, a.nrange = nrange;
    const int s = product<T, false, false>(a, dw, (float*)(ws + pl.part_w), sum_w, st);
    if (s != FF3D_OK) return s;
  }
  if (db) sum_b = sum_job<T>((const float*)(ws + pl.colsum), db, pl.mblocks, 2ll * F);
  const int blocks = sum_x.blocks + sum_w.blocks + sum_b.blocks;
  if (blocks) sum_kernel<T><<<blocks, 256, 0, st>>>(sum_x, sum_w, sum_b);
  return ff3d_launch_status();
}

int check(const void* x, const void* w, const void* h, int64_t ldx, int64_t ldh, int M, int C, int F, int act, int dtype, int pack, const void* ws, int64_t need) {
  FF3D_REQUIRE(x && w && h, FF3D_ERR_NULL);
  FF3D_REQUIRE(dtype == FF3D_F32 || dtype == FF3D_BF16 || dtype == FF3D_F16, FF3D_ERR_BAD_DTYPE);
  FF3D_REQUIRE(M > 0 && M < 0x7fffff00 && C > 0 && F > 0 && ldx >= C && ldh >= F && act >= 0 && act <= 3 && (pack & ~3) == 0, FF3D_ERR_BAD_SHAPE);
  const long long size = dtype == FF3D_F32 ? 4 : 2, per = 16 / size;
  // byte offsets inside a block's rows and inside the weight are 31 bits
  FF3D_REQUIRE(2ll * F * align_up(C, per) * size < 0x7fffffffll && align_up(2ll * F, per) * 256 * size < 0x7fffffffll && ldx * 256 * size < 0x7fffffffll,
               FF3D_ERR_BAD_SHAPE);
  if (!(pack & 1)) FF3D_REQUIRE(C % per == 0 && ldx % per == 0 && ff3d_aligned16(x), FF3D_ERR_ALIGNMENT);
  if (!(pack & 2)) FF3D_REQUIRE(C % per == 0 && ff3d_aligned16(w), FF3D_ERR_ALIGNMENT);
  if (need > 0) FF3D_REQUIRE(ws && ff3d_aligned16(ws), ws ? FF3D_ERR_ALIGNMENT : FF3D_ERR_NULL);
  return FF3D_OK;
}

}  // namespace

extern "C" int64_t ff3d_gated_linear_workspace_bytes(int M, int C, int F, int dtype, int pack, int backward) {
  if (M <= 0 || C <= 0 || F <= 0) return 0;
  if (dtype == FF3D_F32) return plan<float>(M, C, F, pack, backward).total;
  return dtype == FF3D_F16 ? plan<_Float16>(M, C, F, pack, backward).total : plan<__bf16>(M, C, F, pack, backward).total;
}

extern "C" int ff3d_gated_linear_fwd(const void* x, int64_t ldx, const void* weight, const void* bias, void* h, int M, int C, int F, int act,
                                     int dtype, int pack, void* workspace, ff3d_stream_t stream) {
  const int s = check(x, weight, h, ldx, F, M, C, F, act, dtype, pack, workspace, ff3d_gated_linear_workspace_bytes(M, C, F, dtype, pack, 0));
  if (s != FF3D_OK) return s;
  ff3d_clear_error();
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == FF3D_F32) return fwd<float>((const float*)x, ldx, (const float*)weight, (const float*)bias, (float*)h, M, C, F, act, pack, ws, st);
  if (dtype == FF3D_BF16) return fwd<__bf16>((const __bf16*)x, ldx, (const __bf16*)weight, (const __bf16*)bias, (__bf16*)h, M, C, F, act, pack, ws, st);
  return fwd<_Float16>((const _Float16*)x, ldx, (const _Float16*)weight, (const _Float16*)bias, (_Float16*)h, M, C, F, act, pack, ws, st);
}

extern "C" int ff3d_gated_linear_bwd(const void* x, int64_t ldx, const void* weight, const void* bias, const void* dh, int64_t lddh, void* dx, void* dw,
                                     void* db, int M, int C, int F, int act, int dtype, int pack, void* workspace, ff3d_stream_t stream) {
  const int s = check(x, weight, dh, ldx, lddh, M, C, F, act, dtype, pack, workspace, ff3d_gated_linear_workspace_bytes(M, C, F, dtype, pack, 1));
  if (s != FF3D_OK) return s;
  ff3d_clear_error();
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == FF3D_F32)
    return bwd<float>((const float*)x, ldx, (const float*)weight, (const float*)bias, (const float*)dh, lddh, (float*)dx, (float*)dw, (float*)db, M, C, F, act, pack, ws, st);
  if (dtype == FF3D_BF16)
    return bwd<__bf16>((const __bf16*)x, ldx, (const __bf16*)weight, (const __bf16*)bias, (const __bf16*)dh, lddh, (__bf16*)dx, (__bf16*)dw, (__bf16*)db, M, C, F, act, pack, ws, st);
  return bwd<_Float16>((const _Float16*)x, ldx, (const _Float16*)weight, (const _Float16*)bias, (const _Float16*)dh, lddh, (_Float16*)dx, (_Float16*)dw, (_Float16*)db, M, C, F,
                       act, pack, ws, st);
}
