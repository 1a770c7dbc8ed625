// pgk_grad.hip -- CDNA4 (gfx950) kernels for the gradients of a data-parallel
// training step: the global norm over many tensors, clipping, and the
// averaging fold of the ranks' copies (include/pgk.h, pgk_grad_*).
//
//   sumsq   s = sum over all tensors and elements of g^2
//   clip    out = round(c * g),  c = scale * min(1, max_norm / (|scale| sqrt(s) + 1e-6))
//   fold    out = round(scale * (s0 + s1 + ... )),  s = sum of out^2 as stored
//
// Every one of them touches each element once with one to a few operations per
// loaded value, so HBM bounds them (no MFMA, no reuse for LDS to hold) and
// small calls are bound by their launches.
//
// Numerics.  Squares are formed and summed in 64 bits: the square of any f32,
// f16 or bf16 value is exact there and in range (1e30^2, 1e-30^2), and 1e9 terms
// lose nothing a user could see.  The order of the sum is fixed by the sizes and
// the number of CUs, so equal calls give equal bits; there are no atomics.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pgk.h"
#include "pgk_impl.h"

namespace {

#define set_err pgk_set_err

// ---- element types -----------------------------------------------------------

// Wide is what the clip product is formed in: 64 bits where the result keeps
// 24 bits or more (one rounding, to the stored type), 32 bits for a 16-bit result.
template <int DT> struct Type;
template <> struct Type<PGK_DT_DOUBLE> { using T = double; };
template <> struct Type<PGK_DT_F32> { using T = float; };
template <> struct Type<PGK_DT_F16> { using T = _Float16; };
template <> struct Type<PGK_DT_BF16> { using T = __bf16; };

// 16 bytes of T at any element's address: gfx950 loads and stores 16 bytes at
// every alignment, so a tensor may start at any element of a bucket.
template <typename T> constexpr int kWidth = 16 / (int)sizeof(T);
template <typename T, int N> struct Pack { T v[N]; };
template <typename T, int N> using VecT = T __attribute__((ext_vector_type(N)));

template <typename T, int N>
__device__ __forceinline__ void load(T (&x)[N], const T* p) {
  using V = VecT<T, N>;
  typedef V VU __attribute__((aligned(sizeof(T))));
  const V v = *reinterpret_cast<const VU*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = v[i];
}

template <typename T, int N>
__device__ __forceinline__ void store(T* p, const T (&x)[N]) {
  using V = VecT<T, N>;
  typedef V VU __attribute__((aligned(sizeof(T))));
  V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = x[i];
  *reinterpret_cast<VU*>(p) = v;
}

template <typename T>
__device__ __forceinline__ double to_f64(T x) {
  if constexpr (sizeof(T) == 2) return (double)(float)x;
  else return (double)x;
}

// f64 -> the stored type.  A 16-bit result is rounded from 32 bits, one
// instruction each: left to itself the compiler joins the two conversions into
// one that the hardware lacks and spells it out in some 25 integer operations.
template <typename O>
__device__ __forceinline__ O from_f64(double x) {
  if constexpr (sizeof(O) == 2) {
    float f = (float)x;
    asm("" : "+v"(f));
    return (O)f;
  } else {
    return (O)x;
  }
}

// ---- lists of tensors ------------------------------------------------------------

// A launch takes its tensors by value: no table to keep, nothing to copy, and a
// captured graph holds them.  4 KiB of kernel arguments (the runtime adds its own) bound the number.
constexpr int kBlock = 256;
constexpr int kTileVecs = 4;                      // 16-byte vectors per thread and tile
constexpr int kMaxRead = 180;                     // tensors per launch, read only
constexpr int kMaxCopy = 128;                     // tensors per launch, read and written
constexpr int kMaxGrid = PGK_GRAD_WORK_BYTES / 8; // one partial sum per block

template <typename T> constexpr unsigned kTile = kBlock * kTileVecs * kWidth<T>;   // elements

template <int K>
struct ReadList {
  const void* p[K];
  size_t n[K];
  unsigned first[K + 1];                          // tile at which each tensor starts
  int k;
};

template <int K>
struct CopyList {
  const void* p[K];
  void* out[K];
  size_t n[K];
  unsigned first[K + 1];
  int k;
};

// The tensor that tile t lies in, at or after j.
template <typename L>
__device__ __forceinline__ int find(const L& l, unsigned t) {
  int lo = 0, hi = l.k - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (l.first[m] <= t) lo = m; else hi = m - 1;
  }
  return lo;
}

// ---- sums over a block ---------------------------------------------------------

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// The sum over the block, in thread 0.
template <int BLOCK>
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[BLOCK / 64];
  x = wave_sum(x);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x == 0)
#pragma unroll
    for (int w = 1; w < BLOCK / 64; ++w) x += part[w];
  return x;
}

// ---- kernels ---------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(kBlock) void k_grad_sumsq(ReadList<kMaxRead> l, double* parts, int add) {
  constexpr int W = kWidth<T>;
  double acc = 0.0;
  const unsigned tiles = l.first[l.k];
  for (unsigned t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int j = find(l, t);
    const size_t at = (size_t)(t - l.first[j]) * kTile<T>;
    const T* p = (const T*)l.p[j] + at;
    const size_t left = l.n[j] - at;
    for (unsigned e = threadIdx.x * W; e < kTile<T>; e += kBlock * W) {
      if (e + W <= left) {
        T x[W];
        load(x, p + e);
#pragma unroll
        for (int i = 0; i < W; ++i) acc = fma(to_f64(x[i]), to_f64(x[i]), acc);
      } else {
        for (unsigned i = e; i < left; ++i) acc = fma(to_f64(p[i]), to_f64(p[i]), acc);
      }
    }
  }
  acc = block_sum<kBlock>(acc);
  if (threadIdx.x == 0) parts[blockIdx.x] = add ? parts[blockIdx.x] + acc : acc;
}

__global__ __launch_bounds__(1024) void k_grad_finish(const double* parts, int n, double* sumsq) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) acc += parts[i];
  acc = block_sum<1024>(acc);
  if (threadIdx.x == 0) *sumsq = acc;
}

// c, and the norm it is formed from.  Every block forms the same bits.
__device__ __forceinline__ double coefficient(const double* sumsq, int nsum, double scale, double max_norm,
                                              double* norm) {
  double s = 0.0;
  for (int j = 0; j < nsum; ++j) s += sumsq[j];
  *norm = fabs(scale) * sqrt(s);
  const double c = max_norm / (*norm + 1e-6);
  return scale * (c > 1.0 ? 1.0 : c);              // a NaN stays one
}

template <typename O, typename T>
__device__ __forceinline__ O scaled(T x, double c, float cf) {
  if constexpr (sizeof(O) == 2) return (O)((float)x * cf);
  else return (O)(to_f64(x) * c);
}

template <typename T, typename O>
__global__ __launch_bounds__(kBlock) void k_grad_clip(CopyList<kMaxCopy> l, const double* sumsq, int nsum,
                                                      double scale, double max_norm, double* norm) {
  constexpr int W = kWidth<T>;
  double nrm;
  const double c = coefficient(sumsq, nsum, scale, max_norm, &nrm);
  const float cf = (float)c;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = nrm;
  const unsigned tiles = l.first[l.k];
  for (unsigned t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int j = find(l, t);
    const size_t at = (size_t)(t - l.first[j]) * kTile<T>;
    const T* p = (const T*)l.p[j] + at;
    O* o = (O*)l.out[j] + at;
    const size_t left = l.n[j] - at;
    for (unsigned e = threadIdx.x * W; e < kTile<T>; e += kBlock * W) {
      if (e + W <= left) {
        T x[W];
        O y[W];
        load(x, p + e);
#pragma unroll
        for (int i = 0; i < W; ++i) y[i] = scaled<O>(x[i], c, cf);
        store(o + e, y);
      } else {
        for (unsigned i = e; i < left; ++i) o[i] = scaled<O>(p[i], c, cf);
      }
    }
  }
}

constexpr int kMaxSrc = 16;
struct Sources { const void* p[kMaxSrc]; };

template <typename T, typename O>
__global__ __launch_bounds__(kBlock) void k_grad_fold(O* out, Sources src, int nsrc, size_t n, double scale,
                                                      double* parts) {
  constexpr int W = kWidth<T>;
  double sq = 0.0;
  const size_t stride = (size_t)gridDim.x * kBlock * W;
  for (size_t e = ((size_t)blockIdx.x * kBlock + threadIdx.x) * W; e < n; e += stride) {
    if (e + W <= n) {
      double acc[W];
      T x[W];
      load(x, (const T*)src.p[0] + e);
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] = to_f64(x[i]);
      for (int s = 1; s < nsrc; ++s) {
        load(x, (const T*)src.p[s] + e);
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] += to_f64(x[i]);
      }
      O y[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        y[i] = from_f64<O>(acc[i] * scale);
        sq = fma(to_f64(y[i]), to_f64(y[i]), sq);
      }
      store(out + e, y);
    } else {
      for (size_t i = e; i < n; ++i) {
        double acc = to_f64(((const T*)src.p[0])[i]);
        for (int s = 1; s < nsrc; ++s) acc += to_f64(((const T*)src.p[s])[i]);
        const O y = from_f64<O>(acc * scale);
        sq = fma(to_f64(y), to_f64(y), sq);
        out[i] = y;
      }
    }
  }
  if (!parts) return;
  sq = block_sum<kBlock>(sq);
  if (threadIdx.x == 0) parts[blockIdx.x] = sq;
}

// ---- host side ---------------------------------------------------------------------

size_t elem_size(int dt) {
  switch (dt) {
    case PGK_DT_DOUBLE: return 8;
    case PGK_DT_F32: return 4;
    case PGK_DT_F16: case PGK_DT_BF16: return 2;
    default: return 0;
  }
}

bool check_types(const char* what, int dt, int out_dt) {
  if (!elem_size(dt)) { set_err("pgk: %s: bad gradient type %d", what, dt); return false; }
  if (out_dt != dt && !(out_dt == PGK_DT_F32 && elem_size(dt) == 2)) {
    set_err("pgk: %s: output type %d with gradient type %d", what, out_dt, dt);
    return false;
  }
  return true;
}

bool misaligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

bool overlap(const void* p, size_t np, const void* q, size_t nq) {
  const uintptr_t x = (uintptr_t)p, y = (uintptr_t)q;
  return x < y + nq && y < x + np;
}

// The list and every tensor in it: pointers there and on an element, sizes that 64 bits hold.
bool check_list(const char* what, const void* const* p, const size_t* ns, int k, size_t es) {
  if (k < 0 || (k && (!p || !ns))) { set_err("pgk: %s: bad list of %d tensors", what, k); return false; }
  for (int j = 0; j < k; ++j) {
    if (!ns[j]) continue;
    if (!p[j]) { set_err("pgk: %s: NULL tensor %d with n=%zu", what, j, ns[j]); return false; }
    if (misaligned(p[j], es)) { set_err("pgk: %s: tensor %d is not on a multiple of its element size", what, j); return false; }
    if (ns[j] > ((size_t)1 << 40)) { set_err("pgk: %s: tensor %d of %zu elements", what, j, ns[j]); return false; }
  }
  return true;
}

bool check_sums(const char* what, const void* p, const char* name) {
  if (!p || misaligned(p, 8)) { set_err("pgk: %s: %s is NULL or not 8-byte aligned", what, name); return false; }
  return true;
}

int launched(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_err("pgk: %s: launch failed: %s", what, hipGetErrorString(e)); return -1; }
  return 0;
}

unsigned grid_for(size_t tiles) {
  size_t g = (size_t)pgk_cu_count() * 8;
  if (g > (size_t)kMaxGrid) g = kMaxGrid;
  if (tiles < g) g = tiles ? tiles : 1;
  return (unsigned)g;
}

constexpr size_t kMaxTiles = (size_t)1 << 31;      // tile numbers are 32 bits; a launch starts no later tile

template <typename T>
int sumsq_t(const void* const* grads, const size_t* ns, int k, double* sumsq, double* work, hipStream_t s) {
  // how many tiles the fullest launch has: every launch takes the grid that suits it
  size_t most = 0;
  for (int pass = 0; pass < 2; ++pass) {
    ReadList<kMaxRead> l;
    unsigned grid = pass ? grid_for(most) : 0;
    size_t tiles = 0;
    int add = 0;
    l.k = 0;
    for (int j = 0; j <= k; ++j) {
      const size_t more = j < k ? (ns[j] + kTile<T> - 1) / kTile<T> : 0;
      if (l.k && (j == k || l.k == kMaxRead || tiles + more > kMaxTiles)) {
        if (tiles > most) most = tiles;
        if (pass) {
          l.first[l.k] = (unsigned)tiles;
          hipLaunchKernelGGL((k_grad_sumsq<T>), dim3(grid), dim3(kBlock), 0, s, l, work, add);
          if (launched("grad_sumsq")) return -1;
          add = 1;
        }
        l.k = 0;
        tiles = 0;
      }
      if (!more) continue;
      l.p[l.k] = grads[j];
      l.n[l.k] = ns[j];
      l.first[l.k++] = (unsigned)tiles;
      tiles += more;
    }
    if (pass) {
      hipLaunchKernelGGL(k_grad_finish, dim3(1), dim3(1024), 0, s, work, add ? (int)grid : 0, sumsq);
      return launched("grad_sumsq");
    }
  }
  return 0;
}

template <typename T, typename O>
int clip_t(void* const* outs, const void* const* grads, const size_t* ns, int k, const double* sumsq, int nsum,
           double scale, double max_norm, double* norm, hipStream_t s) {
  CopyList<kMaxCopy> l;
  size_t tiles = 0;
  bool any = false;
  l.k = 0;
  for (int j = 0; j <= k; ++j) {
    const size_t more = j < k ? (ns[j] + kTile<T> - 1) / kTile<T> : 0;
    // a launch without tensors still writes the norm
    if ((l.k && (j == k || l.k == kMaxCopy || tiles + more > kMaxTiles)) || (j == k && !any)) {
      l.first[l.k] = (unsigned)tiles;
      hipLaunchKernelGGL((k_grad_clip<T, O>), dim3(grid_for(tiles)), dim3(kBlock), 0, s, l, sumsq, nsum, scale,
                         max_norm, any ? nullptr : norm);
      if (launched("grad_clip")) return -1;
      any = true;
      l.k = 0;
      tiles = 0;
    }
    if (!more) continue;
    l.p[l.k] = grads[j];
    l.out[l.k] = outs[j];
    l.n[l.k] = ns[j];
    l.first[l.k++] = (unsigned)tiles;
    tiles += more;
  }
  return 0;
}

template <typename T, typename O>
int fold_t(void* out, const Sources& src, int nsrc, size_t n, double scale, double* sumsq, double* work,
           hipStream_t s) {
  const unsigned grid = grid_for((n + kBlock * kWidth<T> - 1) / (kBlock * kWidth<T>));
  hipLaunchKernelGGL((k_grad_fold<T, O>), dim3(grid), dim3(kBlock), 0, s, (O*)out, src, nsrc, n, scale,
                     sumsq ? work : nullptr);
  if (launched("grad_fold")) return -1;
  if (!sumsq) return 0;
  hipLaunchKernelGGL(k_grad_finish, dim3(1), dim3(1024), 0, s, work, (int)grid, sumsq);
  return launched("grad_fold");
}

// f(type of the gradients, type of the output) for the pairs check_types lets through.
template <typename F>
int with_types(int dt, int out_dt, F f) {
  switch (dt) {
    case PGK_DT_DOUBLE: return f((double*)nullptr, (double*)nullptr);
    case PGK_DT_F32: return f((float*)nullptr, (float*)nullptr);
    case PGK_DT_F16:
      return out_dt == dt ? f((_Float16*)nullptr, (_Float16*)nullptr) : f((_Float16*)nullptr, (float*)nullptr);
    default:
      return out_dt == dt ? f((__bf16*)nullptr, (__bf16*)nullptr) : f((__bf16*)nullptr, (float*)nullptr);
  }
}

}  // namespace

extern "C" {

int pgk_grad_sumsq(const void* const* grads, const size_t* ns, int k, int dt, double* sumsq, void* work,
                   void* stream) {
  const char* what = "grad_sumsq";
  if (!check_types(what, dt, dt) || !check_list(what, grads, ns, k, elem_size(dt)) ||
      !check_sums(what, sumsq, "sumsq") || !check_sums(what, work, "work")) return -1;
  return with_types(dt, dt, [&](auto* t, auto*) {
    return sumsq_t<std::remove_pointer_t<decltype(t)>>(grads, ns, k, sumsq, (double*)work, (hipStream_t)stream);
  });
}

int pgk_grad_clip(void* const* outs, int out_dt, const void* const* grads, int dt, const size_t* ns, int k,
                  const double* sumsq, int nsum, double scale, double max_norm, double* norm, void* stream) {
  const char* what = "grad_clip";
  if (!check_types(what, dt, out_dt) || !check_list(what, grads, ns, k, elem_size(dt)) ||
      !check_list(what, (const void* const*)outs, ns, k, elem_size(out_dt)) ||
      !check_sums(what, sumsq, "sumsq") || (norm && !check_sums(what, norm, "norm"))) return -1;
  if (nsum < 1) { set_err("pgk: %s: %d partial sums", what, nsum); return -1; }
  if (norm && overlap(norm, 8, sumsq, (size_t)nsum * 8)) { set_err("pgk: %s: norm lies in sumsq", what); return -1; }
  if (!isfinite(scale)) { set_err("pgk: %s: scale %g", what, scale); return -1; }
  if (!(max_norm >= 0)) { set_err("pgk: %s: max_norm %g", what, max_norm); return -1; }
  for (int j = 0; j < k; ++j)
    if (ns[j] && !(outs[j] == grads[j] && dt == out_dt) &&
        overlap(outs[j], ns[j] * elem_size(out_dt), grads[j], ns[j] * elem_size(dt))) {
      set_err("pgk: %s: output %d overlaps its gradient at a different address", what, j);
      return -1;
    }
  return with_types(dt, out_dt, [&](auto* t, auto* o) {
    return clip_t<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>>(
        outs, grads, ns, k, sumsq, nsum, scale, max_norm, norm, (hipStream_t)stream);
  });
}

int pgk_grad_fold(void* out, int out_dt, const void* const* srcs, int nsrc, size_t n, int dt, double scale,
                  double* sumsq, void* work, void* stream) {
  const char* what = "grad_fold";
  if (!check_types(what, dt, out_dt)) return -1;
  if (nsrc < 1 || nsrc > kMaxSrc) { set_err("pgk: %s: nsrc %d outside 1..%d", what, nsrc, kMaxSrc); return -1; }
  if (!isfinite(scale)) { set_err("pgk: %s: scale %g", what, scale); return -1; }
  if (sumsq && (!check_sums(what, sumsq, "sumsq") || !check_sums(what, work, "work"))) return -1;
  const size_t es = elem_size(dt), oes = elem_size(out_dt);
  Sources src{};
  if (n) {
    if (!srcs) { set_err("pgk: %s: NULL list with n=%zu", what, n); return -1; }
    size_t same[kMaxSrc];
    for (int j = 0; j < nsrc; ++j) same[j] = n;
    const void* const o[1] = {out};
    if (!check_list(what, srcs, same, nsrc, es) || !check_list(what, o, same, 1, oes)) return -1;
    for (int j = 0; j < nsrc; ++j) {
      src.p[j] = srcs[j];
      if (!(out == srcs[j] && dt == out_dt) && overlap(out, n * oes, srcs[j], n * es)) {
        set_err("pgk: %s: the output overlaps source %d at a different address", what, j);
        return -1;
      }
    }
  } else if (!sumsq) {
    return 0;
  }
  return with_types(dt, out_dt, [&](auto* t, auto* o) {
    return fold_t<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>>(
        out, src, nsrc, n, scale, sumsq, (double*)work, (hipStream_t)stream);
  });
}

}  // extern "C"
