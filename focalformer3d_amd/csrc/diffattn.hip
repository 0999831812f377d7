// Differential attention, forward and backward, in fp32, bf16 and fp16: per head
//   out = P1 v - lam P2 v,   Pm = softmax_j(scale <q_m, k_m>)       head of q and k: [1 | 2] of d each, of v: 2 d
// and, given dO, with dP = dO v^T (one product serves both maps) and W = P1 - lam P2 (one product for dv):
//   dv = W^T dO,  D1 = rowsum(P1 dP) = <dO, O1>,  D2 = <dO, O2>,  dS1 = P1 (dP - D1),  dS2 = -lam P2 (dP - D2),
//   dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dlam = -sum D2.
// Keys that a boolean mask, a length or the causal order excludes count as absent; a row without keys gives zeros.
//
// The query heads that share a key head are rows of one problem: row = i r + (head within its group), so a block's keys and values
// serve all of them, a single new token fills r columns of a tile, and the gradients of shared heads are summed where they arise.
// Score tiles are 32 x 32 with the long-lived side as columns (queries in the forward and dq kernels, keys in the dk / dv kernel):
// a lane owns half a column of scores, so the softmax statistics of a row are one value per lane, and the tile, rounded, is already
// the operand of the next product (ff3d_mma.h): the weights are rounded once before P v, which makes the error of out 1.06 to 1.45 times that
// of rounding it alone.  Keys and values (queries and dO) pass through LDS once per block in two stages, by
// DMA; their transposed reads use ds_read_b64_tr_b16.
//   forward  one pass with running maximum and sum per map; with few rows the keys are cut into slices that a second kernel joins
//   dq       columns = queries, loops over keys;  dk / dv  columns = keys, loops over the rows.  No atomics: results do not depend
//            on timing.  Scores are recomputed from q, k and the saved reference and sum of each row: the exponent
//            of a large probability is then near zero and exact, where score - log-sum-exp would lose a digit.
// fp16: dS of a long row is far below fp16's normal range, so its columns carry a running power-of-two scale (Scaled).  The forward pass's
// weights are taken times 2^7 or 2^15 (FP16_UP): next to a weight of 1, one below 2^-14 would lose digits and one of 2^-25 vanish, and
// tens of thousands of such keys carry a visible share of a row (10 * 2^-24 each: their sum was off by 4 %).
//
// Measured on one MI355X (large copy 4.77 TB/s, large bf16 product 1309 TFLOP/s):
//   1 x 4096, 16 heads over 4 key heads of 64 columns per map, causal, bf16: forward 184 us (560 TFLOP/s of 2 products of 2 d and 4 d),
//     dq 154, dk / dv 306 .. 312, what comes before and behind them 31.  Bound by the turn of matrix and vector work (two exponentials a pair) in
//     the two waves of a SIMD that the accumulators leave room for (matrix unit 34, 42 and 24 % busy), and in dk / dv by 76 bytes a lane of
//     registers that spill.  fp16: forward 166, backward 590 where bf16 takes 445 (the scales of its columns).
//   4 x 720, 8 heads of 16, fp32, masked: 45, 57, 74 and 12 us.  Bound by splitting the fp32 operands and by the exponentials.
//   8 tokens over 16384 keys, 16 heads over 4 of 64, bf16: 47 us for keys and values at 4.3 TB/s, 5.5 for joining the slices.
#include "ff3d_mma.h"

namespace {

using namespace mma;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int JOIN = 1024;         // most slices of the keys
constexpr int ROWDATA = 6;        // fp32 values per row of the backward pass: reference 1, 2 of the exponentials (log2 units), D1, D2, 1 / sum 1, lam / sum 2

struct Args {
  const char *q, *k, *v, *dout;
  const void* lam;
  const uint8_t* mask;
  const int32_t* lens;
  unsigned* bits;                 // backward: the mask by keys, word (b, i / 32, j) bit i % 32
  long long q_b, q_r, k_b, k_r, v_b, v_r, do_b, do_r;     // elements
  long long m_b, m_r, bits_b;                             // bytes, words
  char *out, *out_rest, *dq, *dk, *dv;
  float *out2, *stat, *part, *rowdata, *d2;
  int B, Nq, Nk, H, G, r, rlog, d, R, Rp, causal, splits, split_len, tiles;   // rlog: log2 r, or -1
  float scale, c;                 // c = scale * log2(e)
};

// the query of a packed row (an integer division costs 25 instructions, and some loops need 32 of them)
__device__ __forceinline__ int query_of(const Args& a, int row) { return a.rlog >= 0 ? row >> a.rlog : row / a.r; }

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Where a column's values are rounded to fp16, they are multiplied by a power of two that keeps the largest so far in [2^9, 2^15];
// the accumulators of the column follow when it changes.  The other types have the exponent range and skip this.
template <typename T>
struct Scaled {
  float s = 0.f;                  // 0: nothing but zeros so far
  template <int N>
  __device__ __forceinline__ void see(float mx, f32x16* acc) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
      mx = max_halves(mx);
      const bool need = mx * s > 32768.f || (s == 0.f && mx > 0.f);
      if (__any(need)) {
        if (need) {
          const int e = (int)((__float_as_uint(mx) >> 23) & 0xff) - 127;
          const float n = ff3d_pow2(9 - e), f = s > 0.f ? n / s : 1.f;
          s = n;
#pragma unroll
          for (int t = 0; t < N; ++t) acc[t] *= f;
        }
      }
    }
  }
  __device__ __forceinline__ float mul() const {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) return s;
    else return 1.f;
  }
  __device__ __forceinline__ float undo() const {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) return s > 0.f ? 1.f / s : 1.f;
    else return 1.f;
  }
};
template <typename T>
__device__ __forceinline__ vec8<T> scaled_frag(const f32x16& c, int step, float mul) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
    vec8<T> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = from_f<T>(c[8 * step + e] * mul);
    return v;
  } else {
    return acc_frag<T>(c, step);
  }
}

// What scaled_frag's rounding left, for a second product.  dS = P (dP - D) sums to nothing over the keys, so what remains of dS K is small
// against its terms, and rounding those once gives dq 1.5 to 2.1 times, dk 1.4 to 2.3 times the error of rounding the result alone (8 or
// 16 columns per map, or few keys).  With the second product it is 1.0 to 1.1 times.  dv is treated alike (1.4 times, and more where few
// weights serve many columns).  It is left out (FINE false) where the products are the bound and the sums are long: see `fine` below.
template <typename T>
__device__ __forceinline__ vec8<T> rest_frag(const f32x16& c, int step, float mul, const vec8<T>& v) {
  vec8<T> r;
  if constexpr (__is_same(T, __bf16)) {              // in pairs, without taking the halves of a register apart
    const u32x4 h = __builtin_bit_cast(u32x4, v);
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = pack_bf16(c[8 * step + 2 * e] - __uint_as_float(h[e] << 16), c[8 * step + 2 * e + 1] - __uint_as_float(h[e] & 0xffff0000u));
    r = __builtin_bit_cast(vec8<T>, w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = from_f<T>(fmaf(c[8 * step + e], mul, -to_f(v[e])));
  }
  return r;
}

// What the rounding of an output left: the backward pass needs <dO, out>, which it takes from every term of a row's sum, to more digits
// than 16 bits hold (with 3 or 4 keys dq's error is 1.1 to 1.2 times that of rounding it, without this 1.6 to 1.7 times)
template <typename T>
__device__ __forceinline__ float rest_of(float x) {
  const float r = x - to_f(from_f<T>(x));
  return fabsf(x) < INFINITY && fabsf(r) < INFINITY ? r : 0.f;       // an output beyond the type's range is what it is
}

// ROWS rows of 2 D elements in LDS, in granules: [map 1 | map 2] of D each (SPLIT; the d of a map may fill only a part) or 2 d elements
template <typename T, int D, int ROWS, int NT, bool SPLIT>
struct Tile {
  static constexpr int P = Type<T>::PER16, GR = 2 * D / P, N = ROWS * GR / NT;
  static_assert(ROWS * GR % NT == 0, "whole granules per thread");
  __device__ __forceinline__ static int source(int g, int d) {         // element offset in a row of the tensor, or -1
    const int e = g * P;
    if constexpr (SPLIT) {
      const int w = e % D;
      return w < d ? (e / D) * d + w : -1;
    } else {
      return e < 2 * d ? e : -1;
    }
  }
  // rows row0 .. of one sequence: row j at base + j * ld (bytes); rows from `limit` on are zeros
  __device__ __forceinline__ static void keys(char* lds, const char* base, long long ld, int row0, int limit, int d, int tid, int wave) {
    const char* p = base + row0 * ld;
    const rsrc_t rs = make_rsrc(p, (long long)(limit - row0) * ld);     // the last row's tail may lie outside: guarded by `limit` below
#pragma unroll
    for (int it = 0; it < N; ++it) {
      const int at = it * NT + tid, r = at / GR, g = place<GR>(r, at % GR), s = source(g, d);
      load_lds16(rs, lds + (it * NT + wave * 64) * 16, row0 + r < limit && s >= 0 ? (unsigned)r * (unsigned)ld + s * (unsigned)sizeof(T) : OUT);
    }
  }
  // packed rows row0 ..: row = i r + h, at base + i * ld + h * head bytes
  __device__ __forceinline__ static void rows(const Args& a, char* lds, const char* base, long long ld, int head, int row0, int d, int tid, int wave) {
    const int i0 = query_of(a, row0);
    const char* p = base + i0 * ld;
    const rsrc_t rs = make_rsrc(p, 0x7fffffff);
#pragma unroll
    for (int it = 0; it < N; ++it) {
      const int at = it * NT + tid, r = at / GR, g = place<GR>(r, at % GR), s = source(g, d);
      const int row = row0 + r, i = query_of(a, row), h = row - i * a.r;
      load_lds16(rs, lds + (it * NT + wave * 64) * 16,
                 row < a.R && s >= 0 ? (unsigned)(i - i0) * (unsigned)ld + (unsigned)h * (unsigned)head + s * (unsigned)sizeof(T) : OUT);
    }
  }
};

// 8 consecutive elements of a row held in registers as an operand (zeros where `in` is false)
template <typename T>
__device__ __forceinline__ vec8<T> load8(const char* p, bool in) {
  vec8<T> v;
  u32x4* w = (u32x4*)&v;
#pragma unroll
  for (int k = 0; k < (int)sizeof(vec8<T>) / 16; ++k) w[k] = in ? *(const u32x4*)(p + 16 * k) : (u32x4)(0u);
  return v;
}

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};
template <typename T>
__device__ __forceinline__ void put4(T* p, float a, float b, float c, float d) {
  Four<T> f = {{from_f<T>(a), from_f<T>(b), from_f<T>(c), from_f<T>(d)}};
  *(Four<T>*)p = f;
}

// The n-th row tile to start.  Under the causal order the last tiles are the longest: they come first, and where all blocks start at
// once, two on a CU, the second of a CU's pair is as short as the first is long.
__device__ __forceinline__ int row_tile(const Args& a, int n) {
  const int first = (int)(gridDim.x <= 512 ? 256 / (gridDim.x / a.tiles) : a.tiles);     // tiles of the first block of every CU
  return n < first ? a.tiles - 1 - n : n - first;
}

__device__ __forceinline__ int key_limit(const Args& a, int b) {
  int n = a.Nk;
  if (a.lens) n = max(0, min(n, a.lens[b]));
  return n;
}

// The mask bytes of a row for a half column of a tile of 32 keys: word q holds keys j0 + 8 q + 4 half .. + 3, as the accumulator does.
struct MaskWords {
  unsigned w[4];
  __device__ __forceinline__ void load(const Args& a, const uint8_t* mrow, int j0, int half) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = j0 + 8 * q + 4 * half;
      if (j + 3 < a.Nk) {
        __builtin_memcpy(&w[q], mrow + j, 4);        // one load, whatever its alignment
      } else {
        w[q] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < a.Nk) w[q] |= (unsigned)mrow[j + e] << (8 * e);
      }
    }
  }
};

// Excludes keys from a 32 x 32 tile with queries as columns: both maps' scores become -inf.
__device__ __forceinline__ void exclude_cols_q(const MaskWords& mask, bool use_mask, f32x16& s1, f32x16& s2, int j0, int jlast, int half) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int j = j0 + 8 * q + 4 * half;
    const unsigned m = use_mask ? mask.w[q] : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e > jlast || (m >> (8 * e) & 0xff)) s1[4 * q + e] = -INFINITY, s2[4 * q + e] = -INFINITY;
  }
}

template <typename T, int D>
__device__ __forceinline__ f32x16 scores(const char* tile, int kb, int map, const Op<T>* other, int lane) {
  constexpr int GR = 2 * D / Type<T>::PER16;
  f32x16 s = (f32x16)(0.f);
#pragma unroll
  for (int st = 0; st < D / 16; ++st) s = mfma_step<T>(op<T>(row_frag<T, GR>(tile, kb * 32 + (lane & 31), map * D + 16 * st, lane >> 5)), other[st], s);
  return s;
}

// waves per SIMD that the registers are cut for: 2 where they fit (two waves hide each other's waits)
constexpr int waves_of(int D, int size, bool fits64) { return size == 4 ? (D <= 16 ? 2 : 1) : (D <= 32 || fits64 ? 2 : 1); }

// ---- forward ------------------------------------------------------------------------------------------------------------------
// ROWS: the 4 waves of a block take 32 rows each and share the keys and values.  Otherwise, where there are few rows, they take the
// same 32 rows and every NW-th tile of 32 keys, with LDS of their own and no barrier, and join what they found at the end.
template <typename T, int D, bool ROWS>
struct FwdShape {
  static constexpr int NW = !ROWS && D == 64 && sizeof(T) == 4 ? 2 : 4, KT = ROWS && sizeof(T) == 2 ? 64 : 32;
  static constexpr int BYTES = KT * (2 * D / Type<T>::PER16) * 16, LDS = (ROWS ? 4 : 4 * NW) * BYTES;
};

template <typename T, int D, bool ROWS, bool MASK>
__global__ __launch_bounds__((FwdShape<T, D, ROWS>::NW * 64), (waves_of(D, sizeof(T), ROWS))) void fwd_kernel(Args a) {
  typedef FwdShape<T, D, ROWS> Shape;
  constexpr int NW = Shape::NW, NT = ROWS ? NW * 64 : 64, KT = Shape::KT, GR = 2 * D / Type<T>::PER16, BYTES = Shape::BYTES;
  constexpr int VT = 2 * D / 32, ST = D / 16, BLOCK_ROWS = ROWS ? NW * 32 : 32;
  // log2 of what the largest weight of a row is taken as: with references up to 2^8 behind (ROWS), 2^15 is the most that any becomes
  constexpr float FP16_UP = sizeof(T) == 2 && !__is_same(T, __bf16) ? (ROWS ? 7.f : 15.f) : 0.f;
  __shared__ __attribute__((aligned(16))) char lds[Shape::LDS];
  __shared__ float found[ROWS ? 1 : NW][4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5;
  const int tid = ROWS ? threadIdx.x : lane, lwave = ROWS ? wave : 0;        // of the waves that load a tile together

  // Blocks go round the 8 XCDs: with the key head running fastest, an XCD works on few of them (their keys and values stay in its L2)
  // and, under the causal order, on long and short tiles alike.
  const int bgs = a.B * a.G, bg = blockIdx.x % bgs, b = bg / a.G, g = bg % a.G, split = blockIdx.x / bgs % a.splits;
  const int tile = row_tile(a, blockIdx.x / bgs / a.splits);
  const int row0 = tile * BLOCK_ROWS + (ROWS ? wave * 32 : 0), row = row0 + (lane & 31);
  const bool in = row < a.R;
  const int rowc = min(row, a.R - 1), i = query_of(a, rowc), h = g * a.r + (rowc - i * a.r);

  Op<T> q[2][ST];
  {
    const char* p = a.q + (b * a.q_b + (long long)i * a.q_r + (long long)h * 2 * a.d) * (long long)sizeof(T);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int e = 16 * st + 8 * half;
        q[m][st] = op<T>(load8<T>(p + (m * a.d + e) * (int)sizeof(T), in && e < a.d));
      }
  }
  const int limit = key_limit(a, b), shift = a.Nk - a.Nq;
  int kend = limit;
  if (a.causal) kend = min(kend, query_of(a, min(a.R - 1, tile * BLOCK_ROWS + BLOCK_ROWS - 1)) + shift + 1);
  const int kbeg = split * a.split_len;
  kend = min(kend, kbeg + a.split_len);
  const int jlast = a.causal ? min(limit - 1, i + shift) : limit - 1;       // last key of this lane's row
  const int wave_first = a.causal ? min(limit - 1, query_of(a, min(row0, a.R - 1)) + shift) : limit - 1;   // smallest in the wave
  const uint8_t* mrow = MASK ? a.mask + b * a.m_b + i * a.m_r : nullptr;

  f32x16 o[2][VT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < VT; ++t) o[m][t] = (f32x16)(0.f);
  float ref[2] = {-INFINITY, -INFINITY}, top[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  MaskWords mask_next;             // of the next 32 keys, asked for one step ahead

  const char* kbase = a.k + (b * a.k_b + (long long)g * 2 * a.d) * (long long)sizeof(T);
  const char* vbase = a.v + (b * a.v_b + (long long)g * 2 * a.d) * (long long)sizeof(T);
  const long long kld = a.k_r * (long long)sizeof(T), vld = a.v_r * (long long)sizeof(T);
  typedef Tile<T, D, KT, NT, true> KTile;
  typedef Tile<T, D, KT, NT, false> VTile;
  const int nt = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;
  constexpr int STRIDE = ROWS ? 1 : NW;
  char* my = lds + (ROWS ? 0 : wave * 4 * BYTES);
  auto stage = [&](int n, int j) {
    KTile::keys(my + (n & 1) * 2 * BYTES, kbase, kld, j, limit, a.d, tid, lwave);
    VTile::keys(my + (n & 1) * 2 * BYTES + BYTES, vbase, vld, j, limit, a.d, tid, lwave);
  };
  const int t0 = ROWS ? 0 : wave;
  if (t0 < nt) {
    stage(0, kbeg + t0 * KT);
    if (MASK) mask_next.load(a, mrow, kbeg + t0 * KT, half);
  }
  for (int t = t0, n = 0; t < nt; t += STRIDE, ++n) {
    const int j0 = kbeg + t * KT;
    const char* kt = my + (n & 1) * 2 * BYTES;
    const char* vt = kt + BYTES;
    if constexpr (ROWS) wait_barrier<0>();
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");        // this wave's own loads, and its reads of the other half
    if (t + STRIDE < nt) stage(n + 1, j0 + STRIDE * KT);
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      const int jb = j0 + kb * 32;
      if (jb >= kend) break;
      const MaskWords mask = mask_next;
      if (MASK) mask_next.load(a, mrow, jb + (ROWS ? 32 : STRIDE * KT), half);
      f32x16 s[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) s[m] = scores<T, D>(kt, kb, m, q[m], lane);
      if (MASK || jb + 31 > wave_first) exclude_cols_q(mask, MASK, s[0], s[1], jb, jlast, half);
      const bool exact = !ROWS || (jb - kbeg) % 128 == 0;
      Op<T> p[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float x = s[m][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) x = fmaxf(x, s[m][e]);
        x = max_halves(x) * a.c;
        // The reference of the exponentials follows the running maximum every fourth step, and at once only where it lies more than 2^8
        // behind.  Following it costs 2 D / 32 accumulators; letting it lag for good (only the 2^8) makes the rounding error of the
        // probabilities 20 % larger, since the largest of them are then spread over a binade instead of sitting just below 1.
        top[m] = fmaxf(top[m], x);
        if (__any(top[m] > ref[m] + (exact ? 0.f : 8.f))) {
          const float n2 = fmaxf(ref[m], top[m]), f = exp2_(ref[m] - (n2 == -INFINITY ? 0.f : n2));
          ref[m] = n2;
          l[m] *= f;
#pragma unroll
          for (int v = 0; v < VT; ++v) o[m][v] *= f;
        }
        const float base = ref[m] == -INFINITY ? 0.f : ref[m] - FP16_UP;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[m][e] = exp2_(fmaf(s[m][e], a.c, -base));
          sum += s[m][e];
        }
        l[m] += sum;
        p[m][0] = op<T>(acc_frag<T>(s[m], 0));
        p[m][1] = op<T>(acc_frag<T>(s[m], 1));
      }
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int v = 0; v < VT; ++v) {
          const Op<T> f = op<T>(col_frag_acc<T, GR>(vt, kb * 32 + 16 * st, v * 32, lane));
          o[0][v] = mfma_step<T>(f, p[0][st], o[0][v]);
          o[1][v] = mfma_step<T>(f, p[1][st], o[1][v]);
        }
    }
  }
  l[0] = sum_halves(l[0]), l[1] = sum_halves(l[1]);

  // what leaves the block: columns e .. e + 3 of O1 and O2 of this lane's row
  float inv[2];
  const float lam = to_f(((const T*)a.lam)[h]);
  const long long at = ((long long)b * a.Nq + i) * a.H + h;
  float* part = a.part + (((long long)split * bgs + bg) * a.R + row) * (4 * a.d + 4);      // [split][bg][row]: O1, O2, references and sums
  auto emit = [&](int e, const float* o1, const float* o2) {
    if (!in || e >= 2 * a.d) return;
    if (a.splits > 1) {
      if (l[0] == 0.f && l[1] == 0.f) return;
      put4(part + e, o1[0], o1[1], o1[2], o1[3]);
      put4(part + 2 * a.d + e, o2[0], o2[1], o2[2], o2[3]);
      return;
    }
    float y[4], z[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = o2[k] * inv[1], y[k] = o1[k] * inv[0] - lam * z[k];
    put4((T*)a.out + at * 2 * a.d + e, y[0], y[1], y[2], y[3]);
    if (a.out2) put4(a.out2 + at * 2 * a.d + e, z[0], z[1], z[2], z[3]);
    if constexpr (sizeof(T) == 2)
      if (a.out_rest) put4((T*)a.out_rest + at * 2 * a.d + e, rest_of<T>(y[0]), rest_of<T>(y[1]), rest_of<T>(y[2]), rest_of<T>(y[3]));
  };
  auto emit_row = [&] {
    if (!in || half) return;
    if (a.splits > 1) {
#pragma unroll
      for (int m = 0; m < 2; ++m) part[4 * a.d + 2 * m] = ref[m] - FP16_UP, part[4 * a.d + 2 * m + 1] = l[m];
    } else if (a.stat) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        a.stat[((long long)bg * 4 + m) * a.R + row] = ref[m] == -INFINITY ? 0.f : ref[m] - FP16_UP;
        a.stat[((long long)bg * 4 + 2 + m) * a.R + row] = inv[m];
      }
    }
  };
  if constexpr (ROWS) {
#pragma unroll
    for (int m = 0; m < 2; ++m) inv[m] = l[m] == 0.f ? 0.f : 1.f / l[m];
#pragma unroll
    for (int v = 0; v < VT; ++v)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float o1[4], o2[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o1[k] = o[0][v][4 * x + k], o2[k] = o[1][v][4 * x + k];
        emit(v * 32 + 8 * x + 4 * half, o1, o2);
      }
    emit_row();
  } else {
    // a wave's sums to LDS; then each takes a share of the elements, weighted by 2^(reference - the largest)
    static_assert(NW * 2 * VT * 16 * 256 <= Shape::LDS, "the sums fit where the keys and values were");
    __syncthreads();
    float* sums = (float*)lds + lane;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      found[wave][m][lane] = ref[m], found[wave][2 + m][lane] = l[m];
#pragma unroll
      for (int v = 0; v < VT; ++v)
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[(((wave * 2 + m) * VT + v) * 16 + e) * 64] = o[m][v][e];
    }
    __syncthreads();
    float w[2][NW];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float r = -INFINITY;
#pragma unroll
      for (int k = 0; k < NW; ++k) r = fmaxf(r, found[k][m][lane]);
      l[m] = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float rk = found[k][m][lane];
        w[m][k] = rk == -INFINITY ? 0.f : exp2_(rk - r);
        l[m] += w[m][k] * found[k][2 + m][lane];
      }
      ref[m] = r;
      inv[m] = l[m] == 0.f ? 0.f : 1.f / l[m];
    }
    for (int it = wave; it < VT * 4; it += NW) {
      const int v = it >> 2, x = it & 3;
      float y[2][4] = {};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int k = 0; k < NW; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[m][e] = fmaf(w[m][k], sums[(((k * 2 + m) * VT + v) * 16 + 4 * x + e) * 64], y[m][e]);
      emit(v * 32 + 8 * x + 4 * half, y[0], y[1]);
    }
    if (wave == 0) emit_row();
  }
}

// joins the slices of the keys: one block per row; 4 d threads per group sum one element of O1 or O2 each over the group's slices
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  __shared__ float wt[2][JOIN], sum[256], norm[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bg = blockIdx.x / a.R, row = blockIdx.x % a.R, b = bg / a.G, g = bg % a.G, i = row / a.r, h = g * a.r + row % a.r;
  const int width = 4 * a.d + 4;
  const long long step = (long long)a.B * a.G * a.R * width;
  const float* p = a.part + (long long)blockIdx.x * width;
  if (wave < 2) {                  // a wave per map: the common reference, each slice's weight and the sum of all
    float top = -INFINITY, l = 0.f;
    for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, p[s * step + 4 * a.d + 2 * wave]);
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    for (int s = lane; s < a.splits; s += 64) {
      const float ls = p[s * step + 4 * a.d + 2 * wave + 1], w = ls == 0.f ? 0.f : exp2_(p[s * step + 4 * a.d + 2 * wave] - top);
      wt[wave][s] = w;
      l = fmaf(w, ls, l);
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
    if (lane == 0) {
      norm[wave] = l == 0.f ? 0.f : 1.f / l;
      if (a.stat) {
        a.stat[((long long)bg * 4 + wave) * a.R + row] = top == -INFINITY ? 0.f : top;
        a.stat[((long long)bg * 4 + 2 + wave) * a.R + row] = l == 0.f ? 0.f : 1.f / l;
      }
    }
  }
  __syncthreads();
  const int w4 = 4 * a.d, e = tid % w4, groups = 256 / w4, m = e >= 2 * a.d;
  float acc = 0.f;
#pragma unroll 8
  for (int s = tid / w4; s < a.splits; s += groups) {
    const float w = wt[m][s];
    if (w != 0.f) acc = fmaf(w, p[s * step + e], acc);      // a slice without keys has written nothing
  }
  sum[tid] = acc;
  __syncthreads();
  if (tid < 2 * a.d) {
    float o1 = 0.f, o2 = 0.f;
    for (int k = 0; k < groups; ++k) o1 += sum[k * w4 + tid], o2 += sum[k * w4 + 2 * a.d + tid];
    const long long to = (((long long)b * a.Nq + i) * a.H + h) * 2 * a.d + tid;
    const float z = o2 * norm[1];
    const float y = o1 * norm[0] - to_f(((const T*)a.lam)[h]) * z;
    ((T*)a.out)[to] = from_f<T>(y);
    if (a.out2) a.out2[to] = z;
    if (sizeof(T) == 2 && a.out_rest) ((T*)a.out_rest)[to] = from_f<T>(rest_of<T>(y));
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------
// Before the products, in one launch: the first row_blocks blocks write the rows' values, the others the mask's words.
// rowdata (B G, ROWDATA, Rp): references of the exponents, D1 = <dO, out> + lam D2, D2 = <dO, O2>, 1 / sum 1, lam / sum 2; zeros behind R, whose
// probabilities are therefore 0.  16 lanes per row.
// Words: 32 queries' mask bytes of a key in one word.  The dk / dv kernel then needs a word or two per lane and step, and can ask for them
// a step ahead (16 byte loads behind the step's DMA, in order, would make it wait for that: 93 instead of 122 us at 4 x 720 x 720, 8 heads
// of 16, fp32, 27 instead of 48 at 3 x 333 x 1777, 4 heads of 32, fp16).
template <typename T>
__global__ __launch_bounds__(256) void prep_kernel(Args a, unsigned row_blocks) {
  if (blockIdx.x >= row_blocks) {
    const int words = (a.Nq + 31) / 32, jt = (a.Nk + 255) / 256;
    const unsigned at = blockIdx.x - row_blocks;
    const int j = (int)(at % jt) * 256 + threadIdx.x, w = (int)(at / jt % words), b = (int)(at / jt / words);
    if (j >= a.Nk) return;
    const uint8_t* p = a.mask + b * a.m_b + j;
    uint8_t v[32];                 // all asked for before the first is looked at
#pragma unroll
    for (int k = 0; k < 32; ++k) v[k] = p[min(w * 32 + k, a.Nq - 1) * a.m_r];
    unsigned bits = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) bits |= v[k] ? 1u << k : 0u;
    a.bits[((long long)b * words + w) * a.Nk + j] = bits;
    return;
  }
  const long long at = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (at >= (long long)a.B * a.G * a.Rp) return;
  const int bg = (int)(at / a.Rp), row = (int)(at % a.Rp), lane = threadIdx.x & 15;
  float v[ROWDATA] = {};
  if (row < a.R) {
    const int b = bg / a.G, g = bg % a.G, i = row / a.r, h = g * a.r + row % a.r;
    const long long o = (((long long)b * a.Nq + i) * a.H + h) * 2 * a.d;
    const T* go = (const T*)a.dout + b * a.do_b + i * a.do_r + (long long)h * 2 * a.d;
    float d = 0.f, d2 = 0.f;
    for (int e = lane; e < 2 * a.d; e += 16) {
      const float x = to_f(go[e]);
      float y = to_f(((const T*)a.out)[o + e]);
      if constexpr (sizeof(T) == 2) y += to_f(((const T*)a.out_rest)[o + e]);
      d = fmaf(x, y, d);
      d2 = fmaf(x, a.out2[o + e], d2);
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) d += __shfl_xor(d, x), d2 += __shfl_xor(d2, x);
    const float lam = to_f(((const T*)a.lam)[h]);
    const float* st = a.stat + (long long)bg * 4 * a.R + row;
    v[0] = st[0], v[1] = st[a.R], v[2] = fmaf(lam, d2, d), v[3] = d2, v[4] = st[2ll * a.R], v[5] = lam * st[3ll * a.R];
  }
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < ROWDATA; ++k) a.rowdata[((long long)bg * ROWDATA + k) * a.Rp + row] = v[k];
}

// Where there are few row tiles, the keys of a row tile are cut into a.splits slices, whose sums go to a.part in fp32
template <typename T, int D, bool MASK, bool FINE>
__global__ __launch_bounds__(256, waves_of(D, sizeof(T), true)) void dq_kernel(Args a) {
  constexpr int NT = 256, KT = sizeof(T) == 2 ? 64 : 32, P = Type<T>::PER16, GR = 2 * D / P, BYTES = KT * GR * 16;
  constexpr int ST = D / 16, VS = 2 * D / 16, QT = D >= 32 ? D / 32 : 1;
  __shared__ __attribute__((aligned(16))) char lds[4 * BYTES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
  const int bgs = a.B * a.G, bg = blockIdx.x % bgs, b = bg / a.G, g = bg % a.G, split = blockIdx.x / bgs % a.splits;
  const int tile = row_tile(a, blockIdx.x / bgs / a.splits);
  const int row = tile * 128 + wave * 32 + (lane & 31);
  const bool in = row < a.R;
  const int rowc = min(row, a.R - 1), i = query_of(a, rowc), h = g * a.r + (rowc - i * a.r);

  Op<T> q[2][ST], go[VS];
  {
    const char* p = a.q + (b * a.q_b + (long long)i * a.q_r + (long long)h * 2 * a.d) * (long long)sizeof(T);
    const char* po = a.dout + (b * a.do_b + (long long)i * a.do_r + (long long)h * 2 * a.d) * (long long)sizeof(T);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int e = 16 * st + 8 * half;
        q[m][st] = op<T>(load8<T>(p + (m * a.d + e) * (int)sizeof(T), in && e < a.d));
      }
#pragma unroll
    for (int st = 0; st < VS; ++st) {
      const int e = 16 * st + 8 * half;
      go[st] = op<T>(load8<T>(po + e * (int)sizeof(T), in && e < 2 * a.d));
    }
  }
  float rd[ROWDATA], rest = 0.f;
#pragma unroll
  for (int k = 0; k < ROWDATA; ++k) rd[k] = a.rowdata[((long long)bg * ROWDATA + k) * a.Rp + rowc];
  const int limit = key_limit(a, b), shift = a.Nk - a.Nq;
  int kend = limit;
  if (a.causal) kend = min(kend, query_of(a, min(a.R - 1, tile * 128 + 127)) + shift + 1);
  int kbeg = 0;
  if (a.splits > 1) {              // whole tiles of the keys that the rows attend
    const int n = kend > 0 ? (kend + KT - 1) / KT : 0;
    kbeg = (int)((long long)n * split / a.splits) * KT;
    kend = min(kend, (int)((long long)n * (split + 1) / a.splits) * KT);
  }
  const int jlast = a.causal ? min(limit - 1, i + shift) : limit - 1;
  const int wave_first = a.causal ? min(limit - 1, query_of(a, min(tile * 128 + wave * 32, a.R - 1)) + shift) : limit - 1;
  const uint8_t* mrow = MASK ? a.mask + b * a.m_b + i * a.m_r : nullptr;

  f32x16 acc[2][QT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < QT; ++t) acc[m][t] = (f32x16)(0.f);
  Scaled<T> sc[2];
  MaskWords mask_next;             // of the next 32 keys, asked for one step ahead

  const char* kbase = a.k + (b * a.k_b + (long long)g * 2 * a.d) * (long long)sizeof(T);
  const char* vbase = a.v + (b * a.v_b + (long long)g * 2 * a.d) * (long long)sizeof(T);
  const long long kld = a.k_r * (long long)sizeof(T), vld = a.v_r * (long long)sizeof(T);
  typedef Tile<T, D, KT, NT, true> KTile;
  typedef Tile<T, D, KT, NT, false> VTile;
  const int nt = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;
  if (nt > 0) {
    KTile::keys(lds, kbase, kld, kbeg, limit, a.d, tid, wave);
    VTile::keys(lds + BYTES, vbase, vld, kbeg, limit, a.d, tid, wave);
    if (MASK) mask_next.load(a, mrow, kbeg, half);
  }
  for (int t = 0; t < nt; ++t) {
    const int j0 = kbeg + t * KT;
    const char* kt = lds + (t & 1) * 2 * BYTES;
    const char* vt = kt + BYTES;
    wait_barrier<0>();
    if (t + 1 < nt) {
      char* nx = lds + ((t + 1) & 1) * 2 * BYTES;
      KTile::keys(nx, kbase, kld, j0 + KT, limit, a.d, tid, wave);
      VTile::keys(nx + BYTES, vbase, vld, j0 + KT, limit, a.d, tid, wave);
    }
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      const int jb = j0 + kb * 32;
      if (jb >= kend) break;
      const MaskWords mask = mask_next;
      if (MASK) mask_next.load(a, mrow, jb + 32, half);
      f32x16 s[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) s[m] = scores<T, D>(kt, kb, m, q[m], lane);
      if (MASK || jb + 31 > wave_first) exclude_cols_q(mask, MASK, s[0], s[1], jb, jlast, half);
      f32x16 dp = (f32x16)(0.f);
#pragma unroll
      for (int st = 0; st < VS; ++st) dp = mfma_step<T>(op<T>(row_frag<T, GR>(vt, kb * 32 + (lane & 31), 16 * st, half)), go[st], dp);
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          // 1 / sum and -lam are factors of the whole column: they wait for the end
          const float ds = exp2_(fmaf(s[m][e], a.c, -rd[m])) * (dp[e] - rd[2 + m]);
          s[m][e] = ds;
          if (m == 1) rest += ds;
          top[m] = fmaxf(top[m], fabsf(ds));
        }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        sc[m].template see<QT>(top[m], acc[m]);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          if constexpr (FINE && D == 64) __builtin_amdgcn_sched_barrier(0);
          const vec8<T> ds = scaled_frag<T>(s[m], st, sc[m].mul());
          const Op<T> f = op<T>(ds);
          Op<T> x[QT];
#pragma unroll
          for (int t = 0; t < QT; ++t) x[t] = op<T>(col_frag_acc<T, GR>(kt, kb * 32 + 16 * st, (D >= 32 ? m * D : 0) + t * 32, lane));
#pragma unroll
          for (int t = 0; t < QT; ++t) acc[m][t] = mfma_step<T>(x[t], f, acc[m][t]);
          if constexpr (FINE) {
            const Op<T> rest = op<T>(rest_frag<T>(s[m], st, sc[m].mul(), ds));
#pragma unroll
            for (int t = 0; t < QT; ++t) acc[m][t] = mfma_step<T>(x[t], rest, acc[m][t]);
            if constexpr (D == 64) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  }
  if (!in) return;
  if (a.d2) {
    // sum_j P2 dP in fp32 = D2 + sum_j P2 (dP - D2): dlam does not carry the rounding of the probabilities that O2 was made of
    rest = sum_halves(rest);
    if (half == 0) a.d2[((long long)split * bgs + bg) * a.Rp + row] = rest;
  }
  if (!a.dq) return;
  const long long at = (((long long)b * a.Nq + i) * a.H + h) * 2 * a.d, all = (long long)a.B * a.Nq * a.H * 2 * a.d;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float f = a.scale * (m == 0 ? rd[4] : -rd[5]) * sc[m].undo();
#pragma unroll
    for (int x = 0; x < QT; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int col = (D >= 32 ? m * D : 0) + x * 32 + 8 * y + 4 * half, w = col % D;
        if (col / D == m && w < a.d) {
          const float o0 = acc[m][x][4 * y] * f, o1 = acc[m][x][4 * y + 1] * f, o2 = acc[m][x][4 * y + 2] * f, o3 = acc[m][x][4 * y + 3] * f;
          if (a.splits > 1) put4(a.part + split * all + at + m * a.d + w, o0, o1, o2, o3);
          else put4((T*)a.dq + at + m * a.d + w, o0, o1, o2, o3);
        }
      }
  }
}

// d = 64 in 16 bits (WIDE): the accumulators of 32 keys take 128 registers, and with the keys and values as operands beside them one wave
// would fill a SIMD alone, its vector and matrix work in turn.  There the block's keys and values stay in LDS, 8 waves share them in
// pairs - one takes the even, one the odd tiles of 32 rows - and the pair's sums are joined at the end.
template <typename T, int D>
constexpr bool wide_v = D == 64 && sizeof(T) == 2;

template <typename T, int D, bool MASK, bool FINE>
__global__ __launch_bounds__((wide_v<T, D> ? 512 : 256), (wide_v<T, D> ? 2 : waves_of(D, sizeof(T), false))) void dkv_kernel(Args a) {
  constexpr bool WIDE = wide_v<T, D>;
  constexpr int NT = WIDE ? 512 : 256, QR = (sizeof(T) == 2 && D != 32) ? 64 : 32, P = Type<T>::PER16, GR = 2 * D / P, BYTES = QR * GR * 16;
  constexpr int RG = ROWDATA * QR / 4, STAGE = 2 * BYTES + (RG + 63) / 64 * 1024;      // RG granules of row values
  constexpr int ST = D / 16, VS = 2 * D / 16, QT = D >= 32 ? D / 32 : 1, VT = 2 * D / 32;
  constexpr int KBYTES = WIDE ? 128 * GR * 16 : 0;   // keys, and values, of the block
  __shared__ __attribute__((aligned(16))) char lds[2 * STAGE + 2 * KBYTES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
  const int bgs = a.B * a.G, bg = blockIdx.x % bgs, b = bg / a.G, g = bg % a.G, split = blockIdx.x / bgs % a.splits;
  const int tile = blockIdx.x / bgs / a.splits;
  const int limit = key_limit(a, b), shift = a.Nk - a.Nq;
  const int kw = wave & 3, jw = tile * 128 + kw * 32, j = jw + (lane & 31);
  const bool in = j < limit;

  const char* kbase = a.k + (b * a.k_b + (long long)g * 2 * a.d) * (long long)sizeof(T);
  const char* vbase = a.v + (b * a.v_b + (long long)g * 2 * a.d) * (long long)sizeof(T);
  const long long kld = a.k_r * (long long)sizeof(T), vld = a.v_r * (long long)sizeof(T);
  char* kt = lds + 2 * STAGE;
  char* vt = kt + KBYTES;
  Op<T> k[2][WIDE ? 1 : ST], v[WIDE ? 1 : VS];
  if constexpr (WIDE) {
    if (tile * 128 < limit) {
      Tile<T, D, 128, NT, true>::keys(kt, kbase, kld, tile * 128, limit, a.d, tid, wave);
      Tile<T, D, 128, NT, false>::keys(vt, vbase, vld, tile * 128, limit, a.d, tid, wave);
    }
  } else {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int e = 16 * st + 8 * half;
        k[m][st] = op<T>(load8<T>(kbase + ((long long)j * a.k_r + m * a.d + e) * (long long)sizeof(T), in && e < a.d));
      }
#pragma unroll
    for (int st = 0; st < VS; ++st) {
      const int e = 16 * st + 8 * half;
      v[st] = op<T>(load8<T>(vbase + ((long long)j * a.v_r + e) * (long long)sizeof(T), in && e < 2 * a.d));
    }
  }
  auto key = [&](int m, int st) {
    if constexpr (WIDE) return op<T>(row_frag<T, GR>(kt, kw * 32 + (lane & 31), m * D + 16 * st, half));
    else return k[m][st];
  };
  auto value = [&](int st) {
    if constexpr (WIDE) return op<T>(row_frag<T, GR>(vt, kw * 32 + (lane & 31), 16 * st, half));
    else return v[st];
  };

  f32x16 dv[VT], dk[2][QT];
#pragma unroll
  for (int t = 0; t < VT; ++t) dv[t] = (f32x16)(0.f);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < QT; ++t) dk[m][t] = (f32x16)(0.f);
  Scaled<T> sv, sk[2];

  const int head = 2 * a.d * (int)sizeof(T);
  const char* qbase = a.q + (b * a.q_b + (long long)g * a.r * 2 * a.d) * (long long)sizeof(T);
  const char* obase = a.dout + (b * a.do_b + (long long)g * a.r * 2 * a.d) * (long long)sizeof(T);
  const long long qld = a.q_r * (long long)sizeof(T), old_ = a.do_r * (long long)sizeof(T);
  const float* rdata = a.rowdata + (long long)bg * ROWDATA * a.Rp;
  typedef Tile<T, D, QR, NT, true> QTile;
  typedef Tile<T, D, QR, NT, false> OTile;
  int rbeg = 0;
  if (a.causal) rbeg = (int)(min((long long)max(0, tile * 128 - shift) * a.r, (long long)a.Rp) / QR * QR);
  int nt = tile * 128 < limit ? (a.R - rbeg + QR - 1) / QR : 0;
  if (a.splits > 1 && nt > 0) {
    const int from = (int)((long long)nt * split / a.splits), to = (int)((long long)nt * (split + 1) / a.splits);
    rbeg += from * QR, nt = to - from;
  }

  auto stage = [&](char* to, int row0) {
    QTile::rows(a, to, qbase, qld, head, row0, a.d, tid, wave);
    OTile::rows(a, to + BYTES, obase, old_, head, row0, a.d, tid, wave);
    if (wave * 64 < RG) {          // QR / 4 granules of each of the arrays
      const rsrc_t rs = make_rsrc(rdata + row0, ((long long)ROWDATA * a.Rp - row0) * 4);
      load_lds16(rs, to + 2 * BYTES + wave * 1024, tid < RG ? (unsigned)(tid / (QR / 4)) * (unsigned)a.Rp * 4u + (tid % (QR / 4)) * 16u : OUT);
    }
  };
  // words of the mask for this lane's key and the queries of a tile's 32 rows: two, since the first query may lie anywhere in a word
  constexpr int SUBS = !MASK || WIDE ? 1 : QR / 32;
  unsigned words[SUBS][2], words_next[SUBS][2];
  const int nwords = (a.Nq + 31) / 32;
  const unsigned* bits = MASK ? a.bits + b * a.bits_b + min(j, a.Nk - 1) : nullptr;
  auto ask = [&](int row0) {
#pragma unroll
    for (int x = 0; x < SUBS; ++x) {
      const int first = row0 + (WIDE ? wave >> 2 : x) * 32, w = query_of(a, min(first, a.R - 1)) >> 5;
      words_next[x][0] = bits[(long long)w * a.Nk];
      words_next[x][1] = bits[(long long)min(w + 1, nwords - 1) * a.Nk];
    }
  };
  if (nt > 0) {
    if constexpr (MASK) ask(rbeg);
    stage(lds, rbeg);
  }
  for (int t = 0; t < nt; ++t) {
    const int row0 = rbeg + t * QR;
    const char* qt = lds + (t & 1) * STAGE;
    const char* ot = qt + BYTES;
    const float* rd = (const float*)(qt + 2 * BYTES);
    wait_barrier<0>();
    if constexpr (MASK) {
#pragma unroll
      for (int x = 0; x < SUBS; ++x) words[x][0] = words_next[x][0], words[x][1] = words_next[x][1];
      if (t + 1 < nt) ask(row0 + QR);
    }
    if (t + 1 < nt) stage(lds + ((t + 1) & 1) * STAGE, row0 + QR);
#pragma unroll
    for (int rb_ = 0; rb_ < (WIDE ? 1 : QR / 32); ++rb_) {
      const int rb = WIDE ? wave >> 2 : rb_;
      // operands are read in groups ahead of the products that use them (a group is waited for once), as far as registers go
      f32x16 s[2] = {(f32x16)(0.f), (f32x16)(0.f)};
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        vec8<T> x[ST];
        Op<T> y[ST];
#pragma unroll
        for (int st = 0; st < ST; ++st) x[st] = row_frag<T, GR>(qt, rb * 32 + (lane & 31), m * D + 16 * st, half), y[st] = key(m, st);
        if constexpr (WIDE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < ST; ++st) s[m] = mfma_step<T>(op<T>(x[st]), y[st], s[m]);
      }
      // (row, key) pairs to leave out: keys past the limit, the causal order, the mask
      const bool some = MASK || jw + 31 >= limit || (a.causal && jw + 31 > query_of(a, row0 + rb * 32) + shift);
      if (some) {
        // one comparison and two selects each, without a branch: keys past the limit lie behind every query's last key
        const int i0 = query_of(a, min(row0 + rb * 32, a.R - 1)), jc = in ? j : 0x7fffffff;
        const unsigned blocked = MASK ? __builtin_amdgcn_alignbit(words[MASK ? rb_ : 0][1], words[MASK ? rb_ : 0][0], i0 & 31) : 0u;   // bit i - i0
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = query_of(a, min(row0 + rb * 32 + acc_row(e, half), a.R - 1));
          const int last = a.causal ? i + shift : 0x7ffffffe;
          const bool no = (jc > last) | (MASK && (blocked >> (i - i0) & 1));
          s[0][e] = no ? -INFINITY : s[0][e];
          s[1][e] = no ? -INFINITY : s[1][e];
        }
      }
      f32x16 dp = (f32x16)(0.f);
#pragma unroll
      for (int st0 = 0; st0 < VS; st0 += 4) {
        constexpr int G = VS < 4 ? VS : 4;
        vec8<T> x[G];
        Op<T> y[G];
#pragma unroll
        for (int st = 0; st < G; ++st) x[st] = row_frag<T, GR>(ot, rb * 32 + (lane & 31), 16 * (st0 + st), half), y[st] = value(st0 + st);
        if constexpr (WIDE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < G; ++st) dp = mfma_step<T>(op<T>(x[st]), y[st], dp);
      }
      // With the keys in LDS 16 rows at a time: their weights and dS are used up before the next ones are formed, which keeps registers free
      // (64 columns with the second products: 371 us in bf16 and 549 in fp16, 1192 and 1133 where all 32 rows' are formed first).  Elsewhere
      // it costs 2 to 10 %.
      constexpr int STEPS = WIDE ? 1 : 2;
#pragma unroll
      for (int s0 = 0; s0 < 2; s0 += STEPS) {
        f32x16 w;                  // elements 8 s0 .. 8 (s0 + STEPS) - 1
        float top[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 2 * s0; y < 2 * (s0 + STEPS); ++y) {
          const int rr = rb * 32 + 8 * y + 4 * half;
          float r4[ROWDATA][4];
#pragma unroll
          for (int n = 0; n < ROWDATA; ++n) *(u32x4*)r4[n] = *(const u32x4*)(rd + n * QR + rr);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int e = 4 * y + x;
            const float p1 = exp2_(fmaf(s[0][e], a.c, -r4[0][x])) * r4[4][x], p2 = exp2_(fmaf(s[1][e], a.c, -r4[1][x])) * r4[5][x];
            w[e] = p1 - p2;
            s[0][e] = p1 * (dp[e] - r4[2][x]);
            s[1][e] = -p2 * (dp[e] - r4[3][x]);
            top[0] = fmaxf(top[0], fabsf(w[e])), top[1] = fmaxf(top[1], fabsf(s[0][e])), top[2] = fmaxf(top[2], fabsf(s[1][e]));
          }
          if constexpr (WIDE) __builtin_amdgcn_sched_barrier(0);
        }
        sv.template see<VT>(top[0], dv);
#pragma unroll
        for (int st = s0; st < s0 + STEPS; ++st) {
          const vec8<T> wv = scaled_frag<T>(w, st, sv.mul());
          const Op<T> f = op<T>(wv);
          vec8<T> x[VT];
#pragma unroll
          for (int t = 0; t < VT; ++t) x[t] = col_frag_acc<T, GR>(ot, rb * 32 + 16 * st, t * 32, lane);
#pragma unroll
          for (int t = 0; t < VT; ++t) dv[t] = mfma_step<T>(op<T>(x[t]), f, dv[t]);
          if constexpr (FINE) {
            const Op<T> rest = op<T>(rest_frag<T>(w, st, sv.mul(), wv));
#pragma unroll
            for (int t = 0; t < VT; ++t) dv[t] = mfma_step<T>(op<T>(x[t]), rest, dv[t]);
          }
        }
        sk[0].template see<QT>(top[1], dk[0]);
        sk[1].template see<QT>(top[2], dk[1]);
#pragma unroll
        for (int st = s0; st < s0 + STEPS; ++st) {
          const vec8<T> ds[2] = {scaled_frag<T>(s[0], st, sk[0].mul()), scaled_frag<T>(s[1], st, sk[1].mul())};
          const Op<T> f[2] = {op<T>(ds[0]), op<T>(ds[1])};
          vec8<T> x[2][QT];        // d = 16: both maps share the columns of one tile
#pragma unroll
          for (int m = 0; m < (D >= 32 ? 2 : 1); ++m)
#pragma unroll
            for (int t = 0; t < QT; ++t) x[m][t] = col_frag_acc<T, GR>(qt, rb * 32 + 16 * st, (D >= 32 ? m * D : 0) + t * 32, lane);
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < QT; ++t) dk[m][t] = mfma_step<T>(op<T>(x[D >= 32 ? m : 0][t]), f[m], dk[m][t]);
          if constexpr (FINE) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const Op<T> rest = op<T>(rest_frag<T>(s[m], st, sk[m].mul(), ds[m]));
#pragma unroll
              for (int t = 0; t < QT; ++t) dk[m][t] = mfma_step<T>(op<T>(x[D >= 32 ? m : 0][t]), rest, dk[m][t]);
            }
          }
        }
      }
    }
  }
  const float fv = sv.undo(), fk[2] = {a.scale * sk[0].undo(), a.scale * sk[1].undo()};
#pragma unroll
  for (int x = 0; x < VT; ++x) dv[x] *= fv;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int x = 0; x < QT; ++x) dk[m][x] *= fk[m];
  if constexpr (WIDE) {            // join the pairs
    float* p = (float*)lds + (kw * (VT + 2 * QT) * 16) * 64 + lane;
    static_assert(4 * (VT + 2 * QT) * 16 * 256 <= (int)sizeof(lds), "the odd waves' sums");
    wait_barrier<0>();             // a block without rows still has its keys on the way to LDS
    if (wave >= 4) {
#pragma unroll
      for (int x = 0; x < VT; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[(x * 16 + e) * 64] = dv[x][e];
#pragma unroll
      for (int x = 0; x < 2 * QT; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[((VT + x) * 16 + e) * 64] = dk[x / QT][x % QT][e];
    }
    __syncthreads();
    if (wave >= 4) return;
#pragma unroll
    for (int x = 0; x < VT; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) dv[x][e] += p[(x * 16 + e) * 64];
#pragma unroll
    for (int x = 0; x < 2 * QT; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) dk[x / QT][x % QT][e] += p[((VT + x) * 16 + e) * 64];
  }
  if (j >= a.Nk) return;           // keys past their sequence's length get zeros
  const long long at = (((long long)b * a.Nk + j) * a.G + g) * 2 * a.d, all = (long long)a.B * a.Nk * a.G * 2 * a.d;
#pragma unroll
  for (int x = 0; x < VT; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int e = x * 32 + 8 * y + 4 * half;
      if (e < 2 * a.d) {
        if (a.splits > 1) put4(a.part + (2ll * split + 1) * all + at + e, dv[x][4 * y], dv[x][4 * y + 1], dv[x][4 * y + 2], dv[x][4 * y + 3]);
        else put4((T*)a.dv + at + e, dv[x][4 * y], dv[x][4 * y + 1], dv[x][4 * y + 2], dv[x][4 * y + 3]);
      }
    }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int x = 0; x < QT; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int col = (D >= 32 ? m * D : 0) + x * 32 + 8 * y + 4 * half, w = col % D;
        if (col / D == m && w < a.d) {
          const float o0 = dk[m][x][4 * y], o1 = dk[m][x][4 * y + 1], o2 = dk[m][x][4 * y + 2], o3 = dk[m][x][4 * y + 3];
          if (a.splits > 1) put4(a.part + 2ll * split * all + at + m * a.d + w, o0, o1, o2, o3);
          else put4((T*)a.dk + at + m * a.d + w, o0, o1, o2, o3);
        }
      }
  }
}

// Behind the products, in one launch: the gradients' slices added in order, and dlam.
// out[i] = sum over the slices of part[slice * step + i]
template <typename T>
struct SumJob {
  const float* part;
  T* out;
  long long n, step;
  int slices, blocks;
};
// dlam[h] = -sum over batch and queries of P2 dP: D2, in 16 bits + (what the dq kernel found beyond it) / sum 2; one block per head, fp64
// sums in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void finish_kernel(Args a, T* dlam, SumJob<T> j0, SumJob<T> j1, SumJob<T> j2) {
  int at = blockIdx.x - (dlam ? a.H : 0);
  if (at >= 0) {
    SumJob<T> j = j0;
    if (at >= j0.blocks) at -= j0.blocks, j = j1;
    if (at >= j.blocks) at -= j.blocks, j = j2;
    for (long long i = ((long long)at * 1024 + threadIdx.x) * 4; i < j.n; i += (long long)j.blocks * 4096) {
      float s[4] = {};
#pragma unroll 8
      for (int k = 0; k < j.slices; ++k) {
        const Four<float> v = *(const Four<float>*)(j.part + k * j.step + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v.v[e];
      }
      put4(j.out + i, s[0], s[1], s[2], s[3]);
    }
    return;
  }
  __shared__ double part[16];
  const int h = blockIdx.x, g = h / a.r, x = h % a.r;
  double s = 0.0;
  const int n = a.B * a.Nq, slices = a.d2 ? a.splits : 0;
  for (int bi = threadIdx.x; bi < n; bi += 1024) {
    const int b = bi / a.Nq, bg = b * a.G + g;
    const long long row = (long long)(bi - b * a.Nq) * a.r + x;
    float rest = 0.f;
#pragma unroll 16
    for (int k = 0; k < slices; ++k) rest += a.d2[((long long)k * a.B * a.G + bg) * a.Rp + row];
    s += (double)a.rowdata[((long long)bg * ROWDATA + 3) * a.Rp + row] + (double)(slices ? rest * a.stat[((long long)bg * 4 + 3) * a.R + row] : 0.f);
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int k = 0; k < 16; ++k) s += part[k];
    dlam[h] = from_f<T>((float)-s);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

struct Split {
  int rows, tiles, splits, len;
};
// Blocks of 128 rows share keys and values among more rows; blocks of 32 rows, whose waves divide the keys, fill the chip where there
// are few.  Where even those leave most of it idle, the keys are cut into slices of at least 512 that a second kernel joins.
Split split_of(const ff3d_diff_attention_t& p) {
  const long long bg = (long long)p.B * p.kv_heads, R = (long long)p.Nq * (p.heads / p.kv_heads);
  Split s;
  s.rows = bg * cdiv(R, 128) >= 256 ? 128 : 32;
  s.tiles = cdiv(R, s.rows);
  const long long blocks = bg * s.tiles;
  long long n = blocks >= 128 ? 1 : cdiv(256, blocks);
  n = n < p.Nk / 512 ? n : p.Nk / 512;
  if (n > JOIN) n = JOIN;
  if (n < 1) n = 1;
  s.len = (int)((cdiv(p.Nk, n) + 127) / 128 * 128);
  s.splits = cdiv(p.Nk, s.len);
  return s;
}

// Backward pass: the loop of a key tile (over rows) or of a row tile (over keys) is cut where the tiles alone leave the chip short of
// blocks, to slices of at least 128 rows or keys; the slices' fp32 sums are added in order.
struct BwdSplit {
  int q, k;
  long long rowdata, d2, bits, dk, total;  // bytes
};
BwdSplit bwd_split_of(const ff3d_diff_attention_t& p) {
  const long long bg = (long long)p.B * p.kv_heads, R = (long long)p.Nq * (p.heads / p.kv_heads);
  auto slices = [](long long blocks, long long len) {
    long long n = blocks >= 384 ? 1 : 512 / blocks;        // two blocks on a CU, and no second round
    n = n < len / 128 ? n : len / 128;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
  };
  BwdSplit s;
  s.q = slices(bg * cdiv(R, 128), p.Nk);
  s.k = slices(bg * cdiv(p.Nk, 128), R);
  s.rowdata = bg * ROWDATA * ((R + 63) / 64 * 64) * 4;
  const long long q = s.q > 1 ? s.q * (long long)p.B * p.Nq * p.heads * 2 * p.d * 4 : 0;
  s.dk = s.k > 1 ? 2ll * s.k * p.B * p.Nk * p.kv_heads * 2 * p.d * 4 : 0;
  s.d2 = s.q * bg * ((R + 63) / 64 * 64) * 4;
  s.bits = p.mask ? ((p.mask_batch ? p.B : 1) * (long long)cdiv(p.Nq, 32) * p.Nk * 4 + 255) / 256 * 256 : 0;
  s.total = s.rowdata + s.d2 + s.bits + s.dk + q;
  return s;
}
inline int sum_grid(long long n) { return (int)(n / 4096 + 1 < 1024 ? n / 4096 + 1 : 1024); }

int check(const ff3d_diff_attention_t* p) {
  FF3D_REQUIRE(p && p->q && p->k && p->v && p->lam, FF3D_ERR_NULL);
  FF3D_REQUIRE(p->dtype == FF3D_F32 || p->dtype == FF3D_BF16 || p->dtype == FF3D_F16, FF3D_ERR_BAD_DTYPE);
  FF3D_REQUIRE(p->B > 0 && p->Nq > 0 && p->Nk > 0 && p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0 && p->scale > 0.f, FF3D_ERR_BAD_SHAPE);
  FF3D_REQUIRE(p->d == 8 || p->d == 16 || p->d == 32 || p->d == 64, FF3D_ERR_UNSUPPORTED);
  const long long r = p->heads / p->kv_heads, size = p->dtype == FF3D_F32 ? 4 : 2, per = 16 / size;
  FF3D_REQUIRE((long long)p->Nq * r < (1ll << 30) && p->Nk < (1 << 30) && (long long)p->B * p->heads < (1ll << 30), FF3D_ERR_BAD_SHAPE);
  const long long w = 2ll * p->d;
  FF3D_REQUIRE(p->q_row >= w * p->heads && p->k_row >= w * p->kv_heads && p->v_row >= w * p->kv_heads, FF3D_ERR_BAD_SHAPE);
  // offsets inside a tile of 128 rows are 31 bits
  FF3D_REQUIRE(p->q_row * size < (1ll << 24) && p->k_row * size < (1ll << 24) && p->v_row * size < (1ll << 24), FF3D_ERR_BAD_SHAPE);
  FF3D_REQUIRE(((p->q_batch | p->q_row | p->k_batch | p->k_row | p->v_batch | p->v_row) % per) == 0, FF3D_ERR_ALIGNMENT);
  FF3D_REQUIRE(ff3d_aligned16(p->q) && ff3d_aligned16(p->k) && ff3d_aligned16(p->v), FF3D_ERR_ALIGNMENT);
  FF3D_REQUIRE(p->q_batch >= 0 && p->k_batch >= 0 && p->v_batch >= 0 && p->mask_batch >= 0 && p->mask_row >= 0, FF3D_ERR_BAD_SHAPE);
  return FF3D_OK;
}

Args args_of(const ff3d_diff_attention_t& p) {
  Args a = {};
  a.q = (const char*)p.q, a.k = (const char*)p.k, a.v = (const char*)p.v, a.lam = p.lam, a.mask = p.mask, a.lens = p.kv_lens;
  a.q_b = p.q_batch, a.q_r = p.q_row, a.k_b = p.k_batch, a.k_r = p.k_row, a.v_b = p.v_batch, a.v_r = p.v_row;
  a.m_b = p.mask_batch, a.m_r = p.mask_row;
  a.B = p.B, a.Nq = p.Nq, a.Nk = p.Nk, a.H = p.heads, a.G = p.kv_heads, a.r = p.heads / p.kv_heads, a.d = p.d, a.causal = p.causal;
  a.rlog = -1;
  for (int k = 0; k < 31; ++k)
    if (a.r == 1 << k) a.rlog = k;
  a.R = a.Nq * a.r, a.Rp = (a.R + 63) / 64 * 64;
  a.scale = p.scale, a.c = p.scale * LOG2E, a.splits = 1, a.split_len = p.Nk;
  return a;
}

template <typename T, int D>
int fwd(const ff3d_diff_attention_t& p, Args a, hipStream_t st) {
  const Split s = split_of(p);
  a.tiles = s.tiles, a.splits = s.splits, a.split_len = s.len;
  const long long blocks = (long long)a.B * a.G * s.tiles * s.splits;
  if (blocks > 0x7fffffffll) return FF3D_ERR_BAD_SHAPE;
  auto kernel = s.rows == 128 ? (a.mask ? fwd_kernel<T, D, true, true> : fwd_kernel<T, D, true, false>)
                              : (a.mask ? fwd_kernel<T, D, false, true> : fwd_kernel<T, D, false, false>);
  kernel<<<(unsigned)blocks, s.rows == 128 ? 256 : FwdShape<T, D, false>::NW * 64, 0, st>>>(a);
  if (s.splits > 1) join_kernel<T><<<(unsigned)((long long)a.B * a.G * a.R), 256, 0, st>>>(a);
  return ff3d_launch_status();
}

template <typename T, int D>
int bwd(const ff3d_diff_attention_t& p, Args a, T* dlam, hipStream_t st) {
  const BwdSplit s = bwd_split_of(p);
  const long long bg = (long long)a.B * a.G, rows = bg * a.Rp, qb = bg * cdiv(a.R, 128) * s.q, kb = bg * cdiv(a.Nk, 128) * s.k;
  if (rows > 0x7fffffffll * 16 || qb > 0x7fffffffll || kb > 0x7fffffffll) return FF3D_ERR_BAD_SHAPE;
  a.d2 = dlam && sizeof(T) == 2 ? a.rowdata + s.rowdata / 4 : nullptr;
  if (a.Nk == 1) a.scale = 0.f;    // the weight of a single key is 1 whatever its score: dq and dk are zero, not the rounding of dP - D
  // The second products of rest_frag cost, at 1 x 4096, 16 heads over 4 of 64, causal: dk / dv 303 -> 371 us and dq 155 -> 192 in bf16,
  // 415 -> 549 and 190 -> 232 in fp16; at 3 x 333 x 1777, 4 heads of 32: +6 and +3 us.  Without them the error is 1.4 to 1.45 times that of
  // one rounding instead of 1.0 at 2200 keys or rows, more where a row attends few keys.  The rule goes by the lengths of the sums alone,
  // over the keys and over the rows of a key head, so that a sequence's gradients have the same accuracy in every batch.
  const bool fine = sizeof(T) == 2 && (D < 64 || (long long)a.R * a.Nk < 1 << 24 || a.R < 1024 || a.Nk < 1024);
  constexpr bool FINE = sizeof(T) == 2, COARSE = sizeof(T) == 2 && D < 64;     // COARSE: the variant where `fine` is false
  a.bits = (unsigned*)(a.rowdata + (s.rowdata + s.d2) / 4);
  a.bits_b = a.m_b ? (long long)cdiv(a.Nq, 32) * a.Nk : 0;
  a.part = a.rowdata + (s.rowdata + s.d2 + s.bits) / 4;
  const long long row_blocks = cdiv(rows, 16), word_blocks = a.mask && a.dk ? (long long)cdiv(a.Nk, 256) * cdiv(a.Nq, 32) * (a.m_b ? a.B : 1) : 0;
  if (row_blocks + word_blocks > 0x7fffffffll) return FF3D_ERR_BAD_SHAPE;
  prep_kernel<T><<<(unsigned)(row_blocks + word_blocks), 256, 0, st>>>(a, (unsigned)row_blocks);
  SumJob<T> dk = {}, dv = {}, dq = {};
  if (a.dk) {
    const long long n = (long long)a.B * a.Nk * a.G * 2 * a.d;
    a.tiles = cdiv(a.Nk, 128), a.splits = s.k;
    auto kernel = fine ? (a.mask ? dkv_kernel<T, D, true, FINE> : dkv_kernel<T, D, false, FINE>)
                       : (a.mask ? dkv_kernel<T, D, true, COARSE> : dkv_kernel<T, D, false, COARSE>);
    kernel<<<(unsigned)kb, wide_v<T, D> ? 512 : 256, 0, st>>>(a);
    if (s.k > 1) dk = {a.part, (T*)a.dk, n, 2 * n, s.k, sum_grid(n)}, dv = {a.part + n, (T*)a.dv, n, 2 * n, s.k, sum_grid(n)};
  }
  a.part += s.dk / 4;
  if (a.dq || a.d2) {
    const long long n = (long long)a.B * a.Nq * a.H * 2 * a.d;
    a.tiles = cdiv(a.R, 128), a.splits = s.q;
    auto kernel = fine ? (a.mask ? dq_kernel<T, D, true, FINE> : dq_kernel<T, D, false, FINE>)
                       : (a.mask ? dq_kernel<T, D, true, COARSE> : dq_kernel<T, D, false, COARSE>);
    kernel<<<(unsigned)qb, 256, 0, st>>>(a);
    if (s.q > 1 && a.dq) dq = {a.part, (T*)a.dq, n, n, s.q, sum_grid(n)};
  }
  const int blocks = (dlam ? a.H : 0) + dk.blocks + dv.blocks + dq.blocks;
  if (blocks) finish_kernel<T><<<blocks, 1024, 0, st>>>(a, dlam, dk, dv, dq);
  return ff3d_launch_status();
}

template <typename T>
int fwd_d(const ff3d_diff_attention_t& p, const Args& a, hipStream_t st) {
  return p.d <= 16 ? fwd<T, 16>(p, a, st) : p.d == 32 ? fwd<T, 32>(p, a, st) : fwd<T, 64>(p, a, st);
}
template <typename T>
int bwd_d(const ff3d_diff_attention_t& p, const Args& a, void* dlam, hipStream_t st) {
  return p.d <= 16 ? bwd<T, 16>(p, a, (T*)dlam, st) : p.d == 32 ? bwd<T, 32>(p, a, (T*)dlam, st) : bwd<T, 64>(p, a, (T*)dlam, st);
}

}  // namespace

extern "C" int64_t ff3d_diff_attention_workspace_bytes(const ff3d_diff_attention_t* p, int backward) {
  if (!p || p->B <= 0 || p->Nq <= 0 || p->Nk <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads) return 0;
  const long long bg = (long long)p->B * p->kv_heads, R = (long long)p->Nq * (p->heads / p->kv_heads);
  if (backward) return bwd_split_of(*p).total;
  const Split s = split_of(*p);
  return s.splits > 1 ? (long long)s.splits * bg * R * (4 * p->d + 4) * 4 : 0;
}

extern "C" int ff3d_diff_attention_fwd(const ff3d_diff_attention_t* p, void* out, float* out2, float* stat, void* out_rest, void* workspace,
                                       ff3d_stream_t stream) {
  const int s = check(p);
  if (s != FF3D_OK) return s;
  FF3D_REQUIRE(out && !out2 == !stat && (p->dtype == FF3D_F32 || !out2 == !out_rest), FF3D_ERR_NULL);
  FF3D_REQUIRE(ff3d_aligned16(out) && ff3d_aligned16(out2) && ff3d_aligned16(out_rest) && ff3d_aligned16(workspace), FF3D_ERR_ALIGNMENT);
  FF3D_REQUIRE(workspace || ff3d_diff_attention_workspace_bytes(p, 0) == 0, FF3D_ERR_NULL);
  ff3d_clear_error();
  Args a = args_of(*p);
  a.out = (char*)out, a.out2 = out2, a.stat = stat, a.out_rest = (char*)out_rest, a.part = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  return p->dtype == FF3D_F32 ? fwd_d<float>(*p, a, st) : p->dtype == FF3D_BF16 ? fwd_d<__bf16>(*p, a, st) : fwd_d<_Float16>(*p, a, st);
}

extern "C" int ff3d_diff_attention_bwd(const ff3d_diff_attention_t* p, const void* out, const float* out2, const float* stat, const void* out_rest,
                                       const void* dout, int64_t dout_batch, int64_t dout_row, void* dq, void* dk, void* dv, void* dlam, void* workspace,
                                       ff3d_stream_t stream) {
  const int s = check(p);
  if (s != FF3D_OK) return s;
  FF3D_REQUIRE(out && out2 && stat && (p->dtype == FF3D_F32 || out_rest) && dout && workspace && (!dk == !dv), FF3D_ERR_NULL);
  const long long size = p->dtype == FF3D_F32 ? 4 : 2;
  FF3D_REQUIRE(dout_row >= 2ll * p->d * p->heads && dout_batch >= 0 && dout_row * size < (1ll << 24), FF3D_ERR_BAD_SHAPE);
  FF3D_REQUIRE((dout_batch | dout_row) % (16 / size) == 0 && ff3d_aligned16(dout) && ff3d_aligned16(dq) && ff3d_aligned16(dk) && ff3d_aligned16(dv) &&
                   ff3d_aligned16(workspace),
               FF3D_ERR_ALIGNMENT);
  // the row values of one sequence are addressed with 31 bits
  FF3D_REQUIRE((long long)ROWDATA * 4 * p->Nq * (p->heads / p->kv_heads) < 0x7fff0000ll, FF3D_ERR_BAD_SHAPE);
  ff3d_clear_error();
  Args a = args_of(*p);
  a.out = (char*)const_cast<void*>(out), a.out2 = const_cast<float*>(out2), a.stat = const_cast<float*>(stat);
  a.out_rest = (char*)const_cast<void*>(out_rest);
  a.dout = (const char*)dout, a.do_b = dout_batch, a.do_r = dout_row, a.dq = (char*)dq, a.dk = (char*)dk, a.dv = (char*)dv, a.rowdata = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  return p->dtype == FF3D_F32 ? bwd_d<float>(*p, a, dlam, st) : p->dtype == FF3D_BF16 ? bwd_d<__bf16>(*p, a, dlam, st) : bwd_d<_Float16>(*p, a, dlam, st);
}
