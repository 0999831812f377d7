// Norm over all elements of many tensors, and clipping by it:
//   n = (sum |g|^2)^(1/2)  |  sum |g|  |  max |g|        out_i = g_i * min(1, max_norm / (n + 1e-6))
// Two passes over the gradients, each one launch for up to TENSORS of them:
//   norm   every block takes one piece of one tensor (pieces are equally long, a block finds its own by bisection of the tensors'
//          first pieces, which travel as kernel arguments: no table in memory, so a call can be captured and costs no copy) and
//          leaves one partial result.  Squares are summed in fp64: the square of any fp32 is exact and cannot overflow there, and
//          the units are idle in a kernel that waits for memory.
//   scale  every block adds all partial results again, in the same order (at most 1024 + one per tensor, a few KB that the caches hold), so there is no third launch and no counter to reset; then scales its piece.  Pieces are taken in
//          the opposite order: the end of the first pass is what the caches still hold.
// Bound by memory: 4 N read, 4 N read again (from the 256 MB cache where the gradients fit it), 4 N written in fp32.
// 88 million fp32 elements: norm 94 us (3.75 TB/s), scale 132 us (5.3 TB/s of both directions); 2.6 million in 35 tensors: 5.2
// and 7.4 us.
#include <algorithm>
#include <new>

#include "ff3d_common.h"

namespace {

constexpr int TENSORS = 120;      // 26 bytes each: the argument block stays under 4 KB
constexpr int THREADS = 256;
enum { KIND_INF = 0, KIND_1 = 1, KIND_2 = 2 };

struct Table {
  const void* src[TENSORS];
  void* dst[TENSORS];
  long long n[TENSORS];
  int first[TENSORS + 1];         // first piece of each tensor
  uint8_t ts[TENSORS], td[TENSORS];
  int count;
};
struct Args {
  long long piece;                // elements of a piece, a multiple of 2048
  double* parts;
  float* norm;
  float max_norm;
  int part0, nparts, kind;        // this launch's first partial result; all of them
};

template <typename T>
struct alignas(16) Pack {
  T v[16 / sizeof(T)];
};

__device__ __forceinline__ double join(double a, double b, int kind) {
  if (kind == KIND_INF) return (b > a || b != b) ? b : a;        // a NaN wins and stays
  return a + b;
}
__device__ __forceinline__ double term(float x, int kind) {
  const double d = (double)x;
  return kind == KIND_2 ? d * d : fabs(d);
}

// joins the block's values; the result is in every thread
__device__ double block_join(double v, int kind, double* lds) {
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) v = join(v, __shfl_xor(v, x), kind);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < THREADS / 64; ++w) v = join(v, lds[w], kind);
  return v;
}

__device__ __forceinline__ int find(const Table& t, int piece) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double norm_piece(const T* p, long long n, int kind) {
  constexpr int P = 16 / sizeof(T);
  double acc = 0.0;
  long long i = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const long long packs = n / P;
    const Pack<T>* q = (const Pack<T>*)p;
    long long k = threadIdx.x;
    for (; k + 3 * THREADS < packs; k += 4 * THREADS) {           // four loads in flight
      Pack<T> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = q[k + u * THREADS];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < P; ++e) acc = join(acc, term((float)v[u].v[e], kind), kind);
    }
    for (; k < packs; k += THREADS) {
      const Pack<T> v = q[k];
#pragma unroll
      for (int e = 0; e < P; ++e) acc = join(acc, term((float)v.v[e], kind), kind);
    }
    i = packs * P;
  }
  for (i += threadIdx.x; i < n; i += THREADS) acc = join(acc, term((float)p[i], kind), kind);
  return acc;
}

__global__ __launch_bounds__(THREADS) void norm_kernel(Table t, Args a) {
  __shared__ double lds[THREADS / 64];
  const int piece = blockIdx.x, k = find(t, piece);
  const long long from = (long long)(piece - t.first[k]) * a.piece, n = min(a.piece, t.n[k] - from);
  double v;
  if (t.ts[k] == FF3D_F32) v = norm_piece((const float*)t.src[k] + from, n, a.kind);
  else if (t.ts[k] == FF3D_BF16) v = norm_piece((const __bf16*)t.src[k] + from, n, a.kind);
  else v = norm_piece((const _Float16*)t.src[k] + from, n, a.kind);
  v = block_join(v, a.kind, lds);
  if (threadIdx.x == 0) a.parts[a.part0 + piece] = v;
}

__device__ __forceinline__ float total(const Args& a, double* lds) {
  double v = 0.0;
  for (int i = threadIdx.x; i < a.nparts; i += THREADS) v = join(v, a.parts[i], a.kind);
  v = block_join(v, a.kind, lds);
  return (float)(a.kind == KIND_2 ? sqrt(v) : v);
}

__global__ __launch_bounds__(THREADS) void total_kernel(Args a) {
  __shared__ double lds[THREADS / 64];
  const float n = total(a, lds);
  if (threadIdx.x == 0) *a.norm = n;
}

template <typename S, typename D>
__device__ __forceinline__ void scale_piece(const S* s, D* d, long long n, float c) {
  constexpr int P = 16 / (sizeof(S) > sizeof(D) ? sizeof(S) : sizeof(D));
  struct alignas(P * sizeof(S)) PS { S v[P]; };
  struct alignas(P * sizeof(D)) PD { D v[P]; };
  long long i = 0;
  if (((reinterpret_cast<uintptr_t>(s) | reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
    const long long packs = n / P;
    long long k = threadIdx.x;
    for (; k + 3 * THREADS < packs; k += 4 * THREADS) {
      PS v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = ((const PS*)s)[k + u * THREADS];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        PD o;
#pragma unroll
        for (int e = 0; e < P; ++e) o.v[e] = (D)((float)v[u].v[e] * c);
        ((PD*)d)[k + u * THREADS] = o;
      }
    }
    for (; k < packs; k += THREADS) {
      const PS v = ((const PS*)s)[k];
      PD o;
#pragma unroll
      for (int e = 0; e < P; ++e) o.v[e] = (D)((float)v.v[e] * c);
      ((PD*)d)[k] = o;
    }
    i = packs * P;
  }
  for (i += threadIdx.x; i < n; i += THREADS) d[i] = (D)((float)s[i] * c);
}

template <typename S>
__device__ __forceinline__ void scale_from(const S* s, void* d, int td, long long from, long long n, float c) {
  if (td == FF3D_F32) scale_piece(s + from, (float*)d + from, n, c);
  else if (td == FF3D_BF16) scale_piece(s + from, (__bf16*)d + from, n, c);
  else scale_piece(s + from, (_Float16*)d + from, n, c);
}

__global__ __launch_bounds__(THREADS) void scale_kernel(Table t, Args a) {
  __shared__ double lds[THREADS / 64];
  const float n = total(a, lds);
  const int piece = gridDim.x - 1 - blockIdx.x, k = find(t, piece);
  if (a.part0 == 0 && piece == 0 && threadIdx.x == 0) *a.norm = n;
  const float q = a.max_norm / (n + 1e-6f), c = q >= 1.f ? 1.f : q;     // a NaN norm makes every output NaN
  if (c == 1.f && t.src[k] == t.dst[k]) return;                         // in place and within the limit: nothing to write
  const long long from = (long long)(piece - t.first[k]) * a.piece, m = min(a.piece, t.n[k] - from);
  if (t.ts[k] == FF3D_F32) scale_from((const float*)t.src[k], t.dst[k], t.td[k], from, m, c);
  else if (t.ts[k] == FF3D_BF16) scale_from((const __bf16*)t.src[k], t.dst[k], t.td[k], from, m, c);
  else scale_from((const _Float16*)t.src[k], t.dst[k], t.td[k], from, m, c);
}

inline bool known(int dt) { return dt == FF3D_F32 || dt == FF3D_BF16 || dt == FF3D_F16; }

// elements of a piece: about 1024 pieces in all, so that four blocks run on each compute unit and the second pass adds few results
long long piece_len(const int64_t* numel, int n) {
  long long total = 0;
  for (int i = 0; i < n; ++i) total += numel[i];
  const long long want = (total + 1023) / 1024;
  return (want + 2047) / 2048 * 2048 > 0 ? (want + 2047) / 2048 * 2048 : 2048;
}

// Whether every output is disjoint from the other outputs and from every gradient but its own (which it may be, whole).  Sorted by
// their first byte, outputs before gradients, a span overlaps an earlier one only if it begins before the furthest end so far.
struct Span {
  uintptr_t from, to;
  int i, grad;
};
int disjoint(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* ts, const int32_t* td, int n) {
  Span* s = new (std::nothrow) Span[2 * (size_t)n];
  if (!s) return FF3D_ERR_LAUNCH;
  int m = 0, status = FF3D_OK;
  for (int i = 0; i < n; ++i)
    if (numel[i] > 0) {
      const uintptr_t a = (uintptr_t)src[i], b = (uintptr_t)dst[i];
      s[m++] = {a, a + numel[i] * (ts[i] == FF3D_F32 ? 4 : 2), i, 1};
      s[m++] = {b, b + numel[i] * (td[i] == FF3D_F32 ? 4 : 2), i, 0};
    }
  std::sort(s, s + m, [](const Span& a, const Span& b) { return a.from != b.from ? a.from < b.from : a.grad < b.grad; });
  uintptr_t grads_to = 0;
  const Span* out = nullptr;
  for (int k = 0; k < m && status == FF3D_OK; ++k) {
    const bool hits = out && s[k].from < out->to;
    if (s[k].grad) {
      if (hits && !(out->i == s[k].i && out->from == s[k].from && out->to == s[k].to)) status = FF3D_ERR_UNSUPPORTED;
      grads_to = std::max(grads_to, s[k].to);
    } else {
      if (hits || s[k].from < grads_to) status = FF3D_ERR_UNSUPPORTED;
      out = s + k;
    }
  }
  delete[] s;
  return status;
}

int run(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* ts, const int32_t* td, int n, int kind, float max_norm, double* parts,
        float* norm, hipStream_t st) {
  FF3D_REQUIRE(n >= 0 && kind >= KIND_INF && kind <= KIND_2, FF3D_ERR_BAD_SHAPE);
  FF3D_REQUIRE(parts && norm && (n == 0 || (src && numel && ts && (!dst || td))), FF3D_ERR_NULL);
  for (int i = 0; i < n; ++i) {
    FF3D_REQUIRE(numel[i] >= 0, FF3D_ERR_BAD_SHAPE);
    FF3D_REQUIRE(known(ts[i]) && (!dst || known(td[i])), FF3D_ERR_BAD_DTYPE);
    FF3D_REQUIRE(numel[i] == 0 || (src[i] && (!dst || dst[i])), FF3D_ERR_NULL);
  }
  if (dst && n > 0) {
    const int s = disjoint(src, dst, numel, ts, td, n);
    if (s != FF3D_OK) return s;
  }
  const long long piece = piece_len(numel, n);
  ff3d_clear_error();
  Args a = {piece, parts, norm, max_norm, 0, 0, kind};
  for (int i = 0; i < n; ++i) a.nparts += (int)((numel[i] + piece - 1) / piece);
  for (int pass = 0; pass < (dst ? 2 : 1); ++pass) {
    a.part0 = 0;
    int i = 0;
    while (i < n) {
      Table t;
      t.count = 0;
      int pieces = 0;
      for (; i < n && t.count < TENSORS; ++i) {
        if (numel[i] == 0) continue;
        const int k = t.count++;
        t.src[k] = src[i], t.dst[k] = dst ? dst[i] : nullptr, t.n[k] = numel[i], t.ts[k] = (uint8_t)ts[i], t.td[k] = dst ? (uint8_t)td[i] : 0;
        t.first[k] = pieces;
        pieces += (int)((numel[i] + piece - 1) / piece);
      }
      if (t.count == 0) break;
      t.first[t.count] = pieces;
      if (pass == 0) norm_kernel<<<pieces, THREADS, 0, st>>>(t, a);
      else scale_kernel<<<pieces, THREADS, 0, st>>>(t, a);
      a.part0 += pieces;
    }
  }
  if (!dst || a.nparts == 0) total_kernel<<<1, THREADS, 0, st>>>(a);
  return ff3d_launch_status();
}

}  // namespace

extern "C" int64_t ff3d_grad_norm_workspace_bytes(const int64_t* numel_host, int n) {
  if (!numel_host || n <= 0) return 8;
  const long long piece = piece_len(numel_host, n);
  long long parts = 1;
  for (int i = 0; i < n; ++i) parts += (numel_host[i] + piece - 1) / piece;
  return parts * 8;
}

extern "C" int ff3d_grad_norm(const void* const* grads_host, const int64_t* numel_host, const int32_t* dtype_host, int n, int kind, void* workspace, float* norm,
                              ff3d_stream_t stream) {
  return run(grads_host, nullptr, numel_host, dtype_host, nullptr, n, kind, 0.f, (double*)workspace, norm, (hipStream_t)stream);
}

extern "C" int ff3d_clip_grads(const void* const* grads_host, void* const* out_host, const int64_t* numel_host, const int32_t* dtype_host,
                               const int32_t* out_dtype_host, int n, int kind, float max_norm, void* workspace, float* norm, ff3d_stream_t stream) {
  FF3D_REQUIRE(n <= 0 || out_host, FF3D_ERR_NULL);
  return run(grads_host, out_host, numel_host, dtype_host, out_dtype_host, n, kind, max_norm, (double*)workspace, norm, (hipStream_t)stream);
}
