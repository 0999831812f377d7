// Gated projection of a feed-forward block, forward and backward, in fp32, bf16 and fp16:
//   h = act(g) * u,   [g | u] = x [Wg ; Wu]^T + [bg | bu]           x (M, C), weight (2 F, C), h (M, F)
// and, given dh:  dg = dh u act'(g),  du = dh act(g),  [dg | du] =: d (M, 2 F),
//   dx = d W,   dW = d^T x,   db = column sums of d.
// All four are matrix products on one tiled kernel with different operand orders and epilogues:
//   gated      both projections in one block: a wave owns the same 32 columns of g and of u, so the activation and the product
//              happen on its accumulators and g, u never reach memory
//   gated_bwd  the same products again with dh in the epilogue -> d (rounded to the type once, as the operand of the two products
//              below has to be) and the column sums of the unrounded d.  g and u are recomputed instead of saved: 2 M C F more
//              multiply-adds, against 2 M F values written and read again and against rounding them, which alone would take the
//              gradients from 1.4 to 1.7 times the error of a single rounding
//   plain      dx and, with its row sum cut into slices that a second kernel adds in order, dW: results do not depend on timing
// A block computes C^T tiles: the n side (features of W, columns of the output) is the row operand, so a lane holds 4 consecutive
// columns of one output row and stores them together.
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
  int vec_out, vec_dh;          // 4-element accesses of out / dh are aligned
  int out_pad;                  // EPI_GATED_BWD: zero columns behind the 2 F
};

// exp for the type: fp32 outputs take the full-precision function, 16-bit ones the hardware's exp2 of the rounded product
template <typename T>
__device__ __forceinline__ float exp_t(float x) {
  if constexpr (sizeof(T) == 4) return expf(x);
  else return __expf(x);
}

template <typename T>
__device__ __forceinline__ float act_f(float g, int act) {
  if (act == ACT_RELU) return g < 0.f ? 0.f : g;               // a NaN stays one
  if (act == ACT_GELU) return g * (0.5f * (1.f + erff(g * 0.70710678118654752f)));
  const float s = 1.f / (1.f + exp_t<T>(-g));
  return act == ACT_SIGMOID ? s : g * s;
}
template <typename T>
__device__ __forceinline__ void act_both(float g, int act, float& a, float& da) {
  if (act == ACT_RELU) {
    a = g < 0.f ? 0.f : g, da = g > 0.f ? 1.f : 0.f;
  } else if (act == ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf, da = cdf + g * exp_t<T>(-0.5f * g * g) * 0.39894228040143268f;
  } else {
    const float s = 1.f / (1.f + exp_t<T>(-g));
    if (act == ACT_SIGMOID) a = s, da = s * (1.f - s);
    else a = g * s, da = s * (1.f + g * (1.f - s));
  }
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

// One operand of a block: ROWS rows (or columns) of it, BK of k per step, DMA-ed into LDS.
// ROW: k is contiguous in memory (row tile), else the rows are (column tile).  DUAL: rows come in blocks of 32 alternating between
// the gate and the value half of the weight.
template <typename T, bool ROW, bool DUAL, int ROWS, int NT>
struct Operand {
  static constexpr int P = Type<T>::PER16, BK = 128 / (int)sizeof(T), N = ROWS * 8 / NT;
  const char *base, *end;
  long long step_bytes;
  unsigned off[N];
  int kk[N];                     // k of the granule inside a step

  __device__ __forceinline__ void init(const char* p, long long bytes, long long ld, int row0, int nrows, int half_rows, long long k0, int tid) {
    end = p + bytes;
    if constexpr (ROW) {
      base = p + (DUAL ? 0 : (long long)row0 * ld * sizeof(T)) + k0 * (long long)sizeof(T);
      step_bytes = 128;
    } else {
      base = p + k0 * ld * (long long)sizeof(T) + (long long)row0 * sizeof(T);
      step_bytes = (long long)BK * ld * sizeof(T);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * NT + tid;
      if constexpr (ROW) {
        const int r = at >> 3, g = place<8>(r, at & 7);
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
  constexpr int BK = 128 / (int)sizeof(T), STEPS = BK / 16, P = Type<T>::PER16;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
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
  A.stage(lds, wave, kn);
  B.stage(lds + ABYTES, wave, kn);
  for (int t = 0; t < nk; ++t) {
    char* cur = lds + (t & 1) * STAGE;
    __syncthreads();               // step t has arrived, and nobody reads the other half any more
    if (t + 1 < nk) {
      char* nxt = lds + ((t + 1) & 1) * STAGE;
      A.stage(nxt, wave, kn - (t + 1) * BK);
      B.stage(nxt + ABYTES, wave, kn - (t + 1) * BK);
    }
    // operands of step s + 1 are read while the matrix unit works on step s
    vec8<T> fa[2][TM], fb[2][TN];
    auto read = [&](int s) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        if constexpr (AROW) fa[s & 1][j] = row_frag<T, 8>(cur, (wm * TM + j) * 32 + (lane & 31), 16 * s, half);
        else fa[s & 1][j] = col_frag<T, BM / P>(cur, 16 * s, (wm * TM + j) * 32, lane);
      }
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        if constexpr (BROW) fb[s & 1][i] = row_frag<T, 8>(cur + ABYTES, (wn * TN + i) * 32 + (lane & 31), 16 * s, half);
        else fb[s & 1][i] = col_frag<T, BN / P>(cur + ABYTES, 16 * s, (wn * TN + i) * 32, lane);
      }
    };
    read(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s + 1 < STEPS) read(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = mfma16(fb[s & 1][i], fa[s & 1][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if constexpr (DUAL) {
    const T* bias = (const T*)p.bias;
    float* sums = (float*)lds;     // EPI_GATED_BWD: column sums of the waves, [WM][2][BNO]
    if constexpr (EPI == EPI_GATED_BWD) __syncthreads();
#pragma unroll
    for (int pr = 0; pr < TN / 2; ++pr)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int nl = (wn * (TN / 2) + pr) * 32 + 8 * q + 4 * half, n = n0 + nl, left = p.N - n;
        float bg[4] = {}, bu[4] = {}, sg[4] = {}, su[4] = {};
        if (bias && left > 0) {
          load4(bias + n, bg, left, false);
          load4(bias + p.F + n, bu, left, false);
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int m = m0 + (wm * TM + j) * 32 + (lane & 31);
          if (m < p.M && left > 0) {
            float g[4], u[4], o[4], o2[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) g[i] = acc[2 * pr][j][4 * q + i] + bg[i], u[i] = acc[2 * pr + 1][j][4 * q + i] + bu[i];
            if constexpr (EPI == EPI_GATED) {
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = act_f<T>(g[i], p.act) * u[i];
              store4((T*)p.out + (long long)m * p.ldo + n, o, left, p.vec_out);
            } else {
              float d[4];
              load4((const T*)p.dh + (long long)m * p.lddh + n, d, left, p.vec_dh);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float a, da;
                act_both<T>(g[i], p.act, a, da);
                o[i] = d[i] * u[i] * da, o2[i] = d[i] * a;
                if (i < left) sg[i] += o[i], su[i] += o2[i];
              }
              T* row = (T*)p.out + (long long)m * p.ldo;
              store4(row + n, o, left, p.vec_out);
              store4(row + p.F + n, o2, left, p.vec_out);
              if (left <= 4)       // the operand of the next products is whole granules wide: zeros behind the 2 F
                for (int i = 0; i < p.out_pad; ++i) row[2 * p.F + i] = from_f<T>(0.f);
            }
          }
        }
        if constexpr (EPI == EPI_GATED_BWD) {
          if (p.colsum) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
              for (int x = 1; x < 32; x <<= 1) sg[i] += __shfl_xor(sg[i], x), su[i] += __shfl_xor(su[i], x);
              if ((lane & 31) == 0) sums[(wm * 2 + 0) * BNO + nl + i] = sg[i], sums[(wm * 2 + 1) * BNO + nl + i] = su[i];
            }
          }
        }
      }
    if constexpr (EPI == EPI_GATED_BWD) {
      if (p.colsum) {
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
  } else {
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
            for (int e = 0; e < 4; ++e) o[e] = acc[i][j][4 * q + e];
            if constexpr (EPI == EPI_PARTIAL) store4((float*)p.out + ((long long)slice * p.M + m) * p.ldo + n, o, left, p.vec_out);
            else store4((T*)p.out + (long long)m * p.ldo + n, o, left, p.vec_out);
          }
        }
      }
  }
}

// out[i] = sum of the slices in order
template <typename T>
__global__ __launch_bounds__(256) void sum_slices_kernel(const float* parts, T* out, int slices, long long n) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float s = 0.f;
    for (int k = 0; k < slices; ++k) s += parts[k * n + i];
    out[i] = from_f<T>(s);
  }
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
  constexpr int LDS = 2 * (BM + BN) * 128;
  auto k = gemm_kernel<T, AROW, BROW, WM, WN, TM, TN, EPI>;
  if (LDS > 64 * 1024) (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  a.mt = cdiv(a.M, BM), a.nt = cdiv(a.N, BNO);
  const long long blocks = (long long)a.mt * a.nt * a.slices;
  if (blocks > 0x7fffffffll) return FF3D_ERR_BAD_SHAPE;
  k<<<(unsigned)blocks, WM * WN * 64, LDS, st>>>(a);
  return ff3d_launch_status();
}

// m rows per block of the gated kernel at these sizes (also the number of partial column sums)
struct Tile {
  int id, bm, bn;
};
template <typename T>
Tile pick(long long M, long long N, bool dual, int slices = 1) {
  const int bn_div = dual ? 2 : 1;
  const Tile t[3] = {{0, 256, 256 / bn_div}, {1, 128, 128 / bn_div}, {2, 64, 128 / bn_div}};
  for (int i = sizeof(T) == 4 ? 1 : 0; i < 2; ++i)
    if ((long long)cdiv(M, t[i].bm) * cdiv(N, t[i].bn) * slices >= 224) return t[i];
  return t[2];
}

template <typename T, bool AROW, bool BROW, int EPI>
int dispatch(const Tile& t, const GemmArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (t.id == 0) return launch<T, AROW, BROW, 2, 4, 4, 2, EPI>(a, st);
  if (t.id <= 1) return launch<T, AROW, BROW, 2, 2, 2, 2, EPI>(a, st);
  return launch<T, AROW, BROW, 2, 2, 1, 2, EPI>(a, st);
}

struct Plan {                    // of one call: packed operands, partial sums, and where they lie in the workspace
  int P, Cp, ldd, slices, kslice, mblocks;
  long long x, w, d, part, colsum, total;
};
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
  p.slices = 1, p.kslice = (int)M, p.mblocks = 0, p.d = p.part = p.colsum = 0;
  if (bwd) {
    p.d = take(M * p.ldd * sizeof(T));
    p.mblocks = cdiv(M, pick<T>(M, F, true).bm);
    p.colsum = take((long long)p.mblocks * 2 * F * 4);
    // dW has few tiles and long sums: cut them until the chip is full, but no shorter than 512 rows
    const int bk = 128 / (int)sizeof(T);
    const long long tiles = (long long)cdiv(2ll * F, 128) * cdiv(C, 128);
    long long s = tiles >= 512 ? 1 : cdiv(512, tiles);
    if (s > M / 512) s = M / 512;
    if (s < 1) s = 1;
    p.kslice = (int)align_up(cdiv(M, s), bk);
    p.slices = cdiv(M, p.kslice);
    p.part = p.slices > 1 ? take((long long)p.slices * 2 * F * C * 4) : 0;
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

inline bool vec_ok(const void* p, long long ld, int size) { return ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * size) == 0; }

template <typename T>
int fwd(const T* x, long long ldx, const T* w, const T* bias, T* h, int M, int C, int F, int act, int pack, char* ws, hipStream_t st) {
  const Plan pl = plan<T>(M, C, F, pack, false);
  long long ldw = C;
  pack_operands<T>(pl, pack, x, ldx, w, ldw, M, C, F, ws, st);
  GemmArgs a = gated_args<T>(x, ldx, w, ldw, bias, M, C, pl.Cp, F, act);
  a.out = h, a.ldo = F, a.vec_out = vec_ok(h, F, sizeof(T));
  return dispatch<T, true, true, EPI_GATED>(pick<T>(M, F, true), a, st);
}

template <typename T>
int bwd(const T* x, long long ldx, const T* w, const T* bias, const T* dh, long long lddh, T* dx, T* dw, T* db, int M, int C, int F, int act,
        int pack, char* ws, hipStream_t st) {
  const Plan pl = plan<T>(M, C, F, pack, true);
  long long ldw = C;
  pack_operands<T>(pl, pack, x, ldx, w, ldw, M, C, F, ws, st);
  T* d = (T*)(ws + pl.d);
  {
    GemmArgs a = gated_args<T>(x, ldx, w, ldw, bias, M, C, pl.Cp, F, act);
    a.out = d, a.ldo = pl.ldd, a.dh = dh, a.lddh = lddh, a.colsum = db ? (float*)(ws + pl.colsum) : nullptr;
    a.out_pad = pl.ldd - 2 * F, a.vec_out = F % 4 == 0, a.vec_dh = vec_ok(dh, lddh, sizeof(T));
    const int s = dispatch<T, true, true, EPI_GATED_BWD>(pick<T>(M, F, true), a, st);
    if (s != FF3D_OK) return s;
  }
  const long long d_bytes = (long long)M * pl.ldd * sizeof(T);
  if (dx) {
    GemmArgs a = {};
    a.a = (const char*)d, a.lda = pl.ldd, a.a_bytes = d_bytes;
    a.b = (const char*)w, a.ldb = ldw, a.b_bytes = ((2ll * F - 1) * ldw + pl.Cp) * (long long)sizeof(T), a.bcols = pl.Cp;
    a.M = M, a.N = C, a.K = 2 * F, a.F = 0, a.slices = 1, a.kslice = (int)align_up(2ll * F, 64);
    a.out = dx, a.ldo = C, a.vec_out = vec_ok(dx, C, sizeof(T));
    const int s = dispatch<T, true, false, EPI_PLAIN>(pick<T>(M, C, false), a, st);
    if (s != FF3D_OK) return s;
  }
  if (dw) {
    GemmArgs a = {};
    a.a = (const char*)d, a.lda = pl.ldd, a.a_bytes = d_bytes, a.acols = pl.ldd;
    a.b = (const char*)x, a.ldb = ldx, a.b_bytes = ((M - 1) * ldx + pl.Cp) * (long long)sizeof(T), a.bcols = pl.Cp;
    a.M = 2 * F, a.N = C, a.K = M, a.slices = pl.slices, a.kslice = pl.kslice, a.ldo = C;
    const Tile t = pick<T>(2ll * F, C, false, pl.slices);
    int s;
    if (pl.slices > 1) {
      a.out = ws + pl.part, a.vec_out = C % 4 == 0;
      s = dispatch<T, false, false, EPI_PARTIAL>(t, a, st);
      if (s == FF3D_OK) sum_slices_kernel<T><<<grid_for(2ll * F * C), 256, 0, st>>>((const float*)(ws + pl.part), dw, pl.slices, 2ll * F * C);
    } else {
      a.out = dw, a.vec_out = vec_ok(dw, C, sizeof(T));
      s = dispatch<T, false, false, EPI_PLAIN>(t, a, st);
    }
    if (s != FF3D_OK) return s;
  }
  if (db) sum_slices_kernel<T><<<grid_for(2ll * F), 256, 0, st>>>((const float*)(ws + pl.colsum), db, pl.mblocks, 2ll * F);
  return ff3d_launch_status();
}

int check(const void* x, const void* w, const void* h, int64_t ldx, int64_t ldh, int M, int C, int F, int act, int dtype, int pack, const void* ws, int64_t need) {
  FF3D_REQUIRE(x && w && h, FF3D_ERR_NULL);
  FF3D_REQUIRE(dtype == FF3D_F32 || dtype == FF3D_BF16 || dtype == FF3D_F16, FF3D_ERR_BAD_DTYPE);
  FF3D_REQUIRE(M > 0 && C > 0 && F > 0 && ldx >= C && ldh >= F && act >= 0 && act <= 3 && (pack & ~3) == 0, FF3D_ERR_BAD_SHAPE);
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
  return dtype == FF3D_F32 ? plan<float>(M, C, F, pack, backward).total : plan<__bf16>(M, C, F, pack, backward).total;
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
