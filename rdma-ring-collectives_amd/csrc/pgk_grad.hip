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
#include <type_traits>

#include "pgk.h"
#include "pgk_impl.h"

namespace {

#define set_err pgk_set_err

// ---- element types -----------------------------------------------------------

// N elements at any element's address, up to 16 bytes: gfx950 loads and stores
// them at every alignment, so a tensor may start at any element of a bucket.
// Non-temporal but where it says otherwise (nothing here is read twice by one launch): a
// read-only pass over 1.3 GB runs at 7.0 TB/s against 6.2 with the default policy,
// a scaled copy of 1.07 GB at 6.4 against 5.85.
template <typename T> constexpr int kWidth = 16 / (int)sizeof(T);

template <bool NT = true, typename T, int N>
__device__ __forceinline__ void load(T (&x)[N], const T* p) {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V VU __attribute__((aligned(sizeof(T))));
  const VU* q = reinterpret_cast<const VU*>(p);
  V v;
  if constexpr (NT) v = __builtin_nontemporal_load(q);
  else v = *q;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = v[i];
}

template <bool NT = true, typename T, int N>
__device__ __forceinline__ void store(T* p, const T (&x)[N]) {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V VU __attribute__((aligned(sizeof(T))));
  V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = x[i];
  if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<VU*>(p));
  else *reinterpret_cast<VU*>(p) = v;
}

// W elements as they lie in memory.  What waits in registers waits like this: the
// compiler would give every element of 16 bits a register of its own, and convert
// what is on its way at once, which means waiting for it.
template <typename T, int W>
struct Raw {
  typedef T Elements __attribute__((ext_vector_type(W)));
  typedef uint32_t Words __attribute__((ext_vector_type(W * sizeof(T) / 4)));
  Words w;
  __device__ __forceinline__ void put(const T (&y)[W]) {
    Elements v;
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = y[i];
    w = __builtin_bit_cast(Words, v);
    asm("" : "+v"(w));
  }
  __device__ __forceinline__ void get(T (&y)[W]) {
    asm("" : "+v"(w));
    const Elements v = __builtin_bit_cast(Elements, w);
#pragma unroll
    for (int i = 0; i < W; ++i) y[i] = v[i];
  }
  __device__ __forceinline__ void load(const T* p) {
    typedef Words WU __attribute__((aligned(2)));
    w = __builtin_nontemporal_load(reinterpret_cast<const WU*>(p));
  }
  __device__ __forceinline__ void store(T* p) const {
    typedef Words WU __attribute__((aligned(2)));
    *reinterpret_cast<WU*>(p) = w;
  }
};

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
// captured graph holds them.  Every further launch costs a small call 3 us and a
// large one 4 to 7, so as many tensors as 4 KiB of kernel arguments can say go
// into one: an address is 48 bits, and one word holds both a tensor's first tile
// and how many elements its last tile has.  A tile is what a block takes at a
// time; every tensor starts one.  A launch takes at most 2^32 elements, a longer
// tensor goes on in the next.
constexpr int kBuckets = 128;

// Outputs that lie as the gradients do (in place, or two flat buffers with equal
// offsets) need no addresses of their own: OWN_OUT says that they have them.
template <bool OWN_OUT> struct OutAddresses {};
template <> struct OutAddresses<true> {
  uint32_t out_lo[218];
  uint32_t out_hi[109];
};

template <bool OWN_OUT>
struct List : OutAddresses<OWN_OUT> {
  static constexpr int kMost = OWN_OUT ? 218 : 351;
  uint32_t lo[kMost], hi[(kMost + 1) / 2];        // addresses: low 32 bits, then 16 more
  uint32_t first[kMost + 1];                      // first tile << kBits | elements in the last tile - 1
  uint32_t where[kBuckets];                       // first tensor in the bucket | last one << 16
  int32_t k, shift;                               // tensors; bucket of a tile: t >> shift
  const char* base;                               // an element of the gradients and
  char* out_base;                                 // the one of the outputs in the same place
};

constexpr int log2_of(unsigned x) { return x > 1 ? 1 + log2_of(x / 2) : 0; }

template <unsigned TILE, bool OWN_OUT>
__host__ __device__ __forceinline__ unsigned tiles_of(const List<OWN_OUT>& l) {
  return l.first[l.k] >> log2_of(TILE);
}

// Where a tile is, and how many elements it has.
template <typename T, typename O>
struct Place {
  const T* p;
  O* o;
  unsigned left;
};

// A block that takes one tile lives for little longer than its loads take, and
// what it waits for before them counts: a search over all tensors, six loads one
// behind the other for 51 of them, added a quarter to a launch (319 against 257
// us for 1.6 GB).  The bucket of a tile leaves none or one of them in most places,
// and what the place is made of is loaded together (the empty asm).  Addresses
// are reached from another one so that the compiler knows them for global memory.
template <unsigned TILE, typename T, typename O, bool OWN_OUT>
__device__ __forceinline__ Place<T, O> find(const List<OWN_OUT>& l, unsigned t) {
  constexpr int kBits = log2_of(TILE);
  const uint32_t both = l.where[t >> l.shift];
  int j = both & 0xffff, top = both >> 16;
  while (j < top) {
    const int m = (j + top + 1) >> 1;
    if (l.first[m] >> kBits <= t) j = m; else top = m - 1;
  }
  const uint32_t first = l.first[j], next = l.first[j + 1], lo = l.lo[j], hi = l.hi[j >> 1];
  uint32_t out_lo = 0, out_hi = 0;
  if constexpr (OWN_OUT) {
    out_lo = l.out_lo[j];
    out_hi = l.out_hi[j >> 1];
  }
  asm volatile("" ::"s"(first), "s"(next), "s"(lo), "s"(hi), "s"(out_lo), "s"(out_hi));
  Place<T, O> r;
  r.left = t + 1 < next >> kBits ? TILE : (first & (TILE - 1)) + 1;
  const size_t at = (size_t)(t - (first >> kBits)) * TILE;
  const int half = 16 * (j & 1);
  const uintptr_t x = (uintptr_t)(hi >> half & 0xffff) << 32 | lo;
  r.p = (const T*)(l.base + (x - (uintptr_t)l.base)) + at;
  if constexpr (OWN_OUT) {
    const uintptr_t y = (uintptr_t)(out_hi >> half & 0xffff) << 32 | out_lo;
    r.o = (O*)(l.out_base + (y - (uintptr_t)l.out_base)) + at;
  } else {
    r.o = (O*)l.out_base + (r.p - (const T*)l.base);
  }
  return r;
}

static_assert(sizeof(List<false>) + 40 <= 4096 && sizeof(List<true>) + 40 <= 4096, "kernel arguments of 4 KiB");

// ---- sums over a block ---------------------------------------------------------

constexpr int kMaxParts = PGK_GRAD_WORK_BYTES / 8;   // one sum per block

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

// A block's share of the sum goes to its own place; the places below `held` have
// the shares of the call's earlier launches in them, the others anything.
template <int BLOCK>
__device__ __forceinline__ void keep(double* parts, int held, double x) {
  x = block_sum<BLOCK>(x);
  if (threadIdx.x == 0) parts[blockIdx.x] = (int)blockIdx.x < held ? parts[blockIdx.x] + x : x;
}

template <typename T, int N>
__device__ __forceinline__ double squares(const T (&x)[N], double acc) {
#pragma unroll
  for (int i = 0; i < N; ++i) acc = fma(to_f64(x[i]), to_f64(x[i]), acc);
  return acc;
}

// ---- sum of squares ----------------------------------------------------------------

// A stream of reads, 16 bytes x UNROLL in flight per thread; the f64 conversions
// and products hide behind it (accumulating in 32 bits takes the same time).
// NT: what does not fit the 256 MiB Infinity Cache is read past it.  What does is
// left there for the clip that follows: both together take 33 against 39 us for
// 75 MiB, 66 against 74 for 150 MiB, the norm alone 14.7 against 13.6 for 75 MiB.
template <typename T, int BLOCK, int UNROLL, bool NT>
__global__ __launch_bounds__(BLOCK) void k_grad_sumsq(List<false> l, unsigned grid, double* parts, int held) {
  constexpr int W = kWidth<T>;
  constexpr unsigned kTile = BLOCK * UNROLL * W;
  double acc = 0.0;
  const unsigned tiles = tiles_of<kTile>(l);
  for (unsigned t = blockIdx.x; t < tiles; t += grid) {
    const Place<T, T> at = find<kTile, T, T>(l, t);
    const T* p = at.p;
    const unsigned left = at.left;
    if (left == kTile) {
      T x[UNROLL][W];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) load<NT>(x[u], p + (u * BLOCK + threadIdx.x) * W);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) acc = squares(x[u], acc);
    } else {
      for (unsigned e = threadIdx.x * W; e < left; e += BLOCK * W) {
        if (e + W <= left) {
          T x[W];
          load<NT>(x, p + e);
          acc = squares(x, acc);
        } else {
          for (unsigned i = e; i < left; ++i) acc = fma(to_f64(p[i]), to_f64(p[i]), acc);
        }
      }
    }
  }
  keep<BLOCK>(parts, held, acc);
}

constexpr int kFinishBlock = 1024;
__global__ __launch_bounds__(kFinishBlock) void k_grad_finish(const double* parts, int n, double* sumsq) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += kFinishBlock) acc += parts[i];
  acc = block_sum<kFinishBlock>(acc);
  if (threadIdx.x == 0) *sumsq = acc;
}

// ---- clip --------------------------------------------------------------------------

// c, and the norm it is formed from, in every lane of a wave.
__device__ __forceinline__ double coefficient(const double* sumsq, int nsum, double scale, double max_norm,
                                              double* norm) {
  double s = 0.0;
  if (nsum == 1) {
    s = sumsq[0];
  } else {
    for (int j = threadIdx.x & 63; j < nsum; j += 64) s += sumsq[j];
    s = wave_sum(s);
  }
  *norm = fabs(scale) * sqrt(s);
  const double c = max_norm / (*norm + 1e-6);
  return c > 1.0 || isinf(max_norm) ? scale : scale * c;   // a NaN of the norm's stays one
}

// One tile per block: blocks that come and go keep reads and writes mixed (a grid
// that loops streams 10-15% slower).  A vector is 16 bytes of the wider type: a
// lane that stores two halves of 32 bytes leaves every store instruction with gaps
// (5.4 against 6.5 TB/s).  Blocks of 256 threads with a vector each lead where the
// types are equal (368M f32: 451 us, with two vectors 476, 512 threads 464, 1024
// threads 478), with two each where the output is wider, whose reads are of 8 bytes
// (267M bf16: 252 us, one vector 276, 1024 threads with one 262).
constexpr int kClipBlock = 256;
template <typename T, typename O> constexpr int kClipVecs = sizeof(O) > sizeof(T) ? 2 : 1;
template <typename T, typename O> constexpr unsigned kClipTile = kClipBlock * kWidth<O> * kClipVecs<T, O>;

// One wave of a block forms c while the block's loads are on their way; the others
// wait for it rather than do the 64-bit root and quotient as well.
template <typename T, typename O, bool OWN_OUT>
__global__ __launch_bounds__(kClipBlock) void k_grad_clip(List<OWN_OUT> l, const double* sumsq, int nsum,
                                                          double scale, double max_norm, double* norm) {
  constexpr int W = kWidth<O>, U = kClipVecs<T, O>;
  __shared__ double shared_c;
  const Place<T, O> at = find<kClipTile<T, O>, T, O>(l, blockIdx.x);
  const T* p = at.p;
  O* o = at.o;
  Raw<T, W> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned e = (u * kClipBlock + threadIdx.x) * W;
    if (e + W <= at.left) raw[u].load(p + e);      // on its way while c is formed
  }
  if (threadIdx.x < 64) {
    double nrm;
    const double c = coefficient(sumsq, nsum, scale, max_norm, &nrm);
    if (threadIdx.x == 0) {
      shared_c = c;
      if (norm && blockIdx.x == 0) *norm = nrm;
    }
  }
  __syncthreads();
  const double c = shared_c;
  // in place, a step that is not clipped needs no writes
  if constexpr (std::is_same_v<T, O>)
    if (o == p && c == 1.0) return;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned e = (u * kClipBlock + threadIdx.x) * W;
    if (e + W <= at.left) {
      T x[W];
      O y[W];
      raw[u].get(x);
#pragma unroll
      for (int i = 0; i < W; ++i) y[i] = from_f64<O>(to_f64(x[i]) * c);
      store(o + e, y);
    } else {
      for (unsigned i = e; i < at.left; ++i) o[i] = from_f64<O>(to_f64(p[i]) * c);
    }
  }
}

// The norm alone, where there are no elements.
__global__ __launch_bounds__(64) void k_grad_norm(const double* sumsq, int nsum, double scale, double* norm) {
  double nrm;
  coefficient(sumsq, nsum, scale, 0.0, &nrm);
  if (threadIdx.x == 0) *norm = nrm;
}

// ---- averaging fold ------------------------------------------------------------------

constexpr int kMaxSrc = 16;
constexpr int kMaxUnrolled = 8;                   // sources whose loads are all in flight at once
struct Sources { const void* p[kMaxSrc]; };

// The mean of W elements at e, summed left to right; its squares into sq.
template <typename T, typename O, int NS, int W>
__device__ __forceinline__ void fold(O (&y)[W], const Sources& src, int nsrc, size_t e, double scale, double* sq) {
  T x[NS][W];
#pragma unroll
  for (int s = 0; s < NS; ++s) load(x[s], (const T*)src.p[s] + e);
  double acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = to_f64(x[0][i]);
#pragma unroll
  for (int s = 1; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] += to_f64(x[s][i]);
  if constexpr (NS == kMaxUnrolled) {
#pragma unroll 4
    for (int s = NS; s < nsrc; ++s) {
      T z[W];
      load(z, (const T*)src.p[s] + e);
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] += to_f64(z[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) y[i] = from_f64<O>(acc[i] * scale);
  *sq = squares(y, *sq);
}

template <typename T, typename O>
__device__ __forceinline__ O fold_one(const Sources& src, int nsrc, size_t e, double scale, double* sq) {
  double acc = to_f64(((const T*)src.p[0])[e]);
  for (int s = 1; s < nsrc; ++s) acc += to_f64(((const T*)src.p[s])[e]);
  const O y = from_f64<O>(acc * scale);
  *sq = fma(to_f64(y), to_f64(y), *sq);
  return y;
}

// Elements [e0, e1), a vector per thread at a time, in a grid of at most as many
// blocks as the workspace holds sums of.  Blocks of 1024 threads lose least by
// that: 85 us for 3 f32 sources of 30M elements (256 threads 92), 107 us for 4 f16
// sources of 50M to f32 (118); fetching the next vectors ahead makes it slower.
// The output is stored with the default policy, for what reads it next: the 30M
// elements take 85 us, with a clip behind 114; past the caches 79 and 120.  An output
// of 600 MiB takes 344 and 507, past the caches 324 and 518.
constexpr int kFoldBlock = 1024;
template <typename T, typename O, int NS>
__global__ __launch_bounds__(kFoldBlock) void k_grad_fold(O* out, Sources src, int nsrc, size_t e0, size_t e1,
                                                          double scale, double* parts, int held) {
  constexpr int W = kWidth<O>;
  double sq = 0.0;
  for (size_t e = e0 + ((size_t)blockIdx.x * kFoldBlock + threadIdx.x) * W; e < e1;
       e += (size_t)gridDim.x * kFoldBlock * W) {
    if (e + W <= e1) {
      O y[W];
      fold<T, O, NS>(y, src, nsrc, e, scale, &sq);
      store<false>(out + e, y);
    } else {
      for (size_t i = e; i < e1; ++i) out[i] = fold_one<T, O>(src, nsrc, i, scale, &sq);
    }
  }
  if (parts) keep<kFoldBlock>(parts, held, sq);
}

// The burst form of pgk_reduce_multi (pgk_reduce.hip) for gradients: every
// thread folds TILES vectors, reads only, and stores them at the end, so the
// chip reads and then writes.  8 sources x 64 MiB of equal types, called one behind
// the other: 95.3 us (6.3 TB/s) against 110 a vector at a time (f32 95.0, 106.6); the
// sum is 2.2 us of it.  (rocprofv3 traces the kernel at 111 us; no timing outside it,
// in a row or alone, shows that.)  It does not pay below 5 sources (4 of 64 MiB 58.5
// against 57.2, 2 51 against 37.5), nor where the output is wider (8 bf16 sources to
// f32 126 against 117, 4 f16 sources 138 against 107).
constexpr int kBurstBlock = 256;
template <typename T, int NS, int TILES>
__global__ __launch_bounds__(kBurstBlock) void k_grad_fold_burst(T* out, Sources src, size_t e0, size_t e1,
                                                                 double scale, double* parts, int held) {
  constexpr int W = kWidth<T>;
  const size_t base = e0 + ((size_t)blockIdx.x * (kBurstBlock * TILES) + threadIdx.x) * W;
  double sq = 0.0;
  Raw<T, W> held_y[TILES];                        // 16 bytes each: 128 registers for 32
#pragma unroll
  for (int u = 0; u < TILES; ++u) {
    const size_t e = base + (size_t)u * (kBurstBlock * W);
    if (e < e1) {
      T y[W];
      fold<T, T, NS>(y, src, NS, e, scale, &sq);
      held_y[u].put(y);
    }
  }
  asm volatile("" ::: "memory");                  // no store is scheduled among the loads
#pragma unroll
  for (int u = 0; u < TILES; ++u) {
    const size_t e = base + (size_t)u * (kBurstBlock * W);
    if (e < e1) held_y[u].store(out + e);
  }
  if (parts) keep<kBurstBlock>(parts, held, sq);
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
    if ((uintptr_t)p[j] >> 48) { set_err("pgk: %s: tensor %d: %p is no device address", what, j, p[j]); return false; }
    if (ns[j] > ((size_t)1 << 40)) { set_err("pgk: %s: tensor %d of %zu elements", what, j, ns[j]); return false; }
  }
  return true;
}

bool check_sums(const char* what, const void* p, const char* name) {
  if (!p || misaligned(p, 8)) { set_err("pgk: %s: %s is NULL or not 8-byte aligned", what, name); return false; }
  return true;
}

bool check_work(const char* what, const double* sumsq, const void* work) {
  if (!check_sums(what, sumsq, "sumsq") || !check_sums(what, work, "work")) return false;
  if (overlap(sumsq, 8, work, PGK_GRAD_WORK_BYTES)) { set_err("pgk: %s: sumsq lies in work", what); return false; }
  return true;
}

// Whether a result's or the workspace's place lies in none of the tensors: kernels that
// read or write them are on their way while it is written.
bool check_apart(const char* what, const char* name, const void* p, size_t bytes, const void* const* ts,
                 const size_t* ns, int k, size_t es) {
  for (int j = 0; j < k; ++j)
    if (ns[j] && overlap(p, bytes, ts[j], ns[j] * es)) { set_err("pgk: %s: %s lies in tensor %d", what, name, j); return false; }
  return true;
}

int launched(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_err("pgk: %s: launch failed: %s", what, hipGetErrorString(e)); return -1; }
  return 0;
}

// Fills the buckets of a list that is complete.
template <unsigned TILE, bool OWN_OUT>
void index(List<OWN_OUT>& l) {
  const unsigned tiles = tiles_of<TILE>(l);
  l.shift = 0;
  while ((tiles - 1) >> l.shift >= (unsigned)kBuckets) ++l.shift;
  int j = 0;
  auto holds = [&](uint64_t t) {                  // the tensor that tile t lies in, or the last one
    while (j + 1 < l.k && l.first[j + 1] >> log2_of(TILE) <= t) ++j;
    return (uint32_t)j;
  };
  for (unsigned b = 0; b < (unsigned)kBuckets; ++b) {
    const uint32_t first = holds((uint64_t)b << l.shift);
    l.where[b] = first | holds((((uint64_t)b + 1) << l.shift) - 1) << 16;
  }
}

inline void put_address(uint32_t* lo, uint32_t* hi, int j, const void* p) {
  const uintptr_t x = (uintptr_t)p;
  lo[j] = (uint32_t)x;
  hi[j >> 1] = j & 1 ? hi[j >> 1] | (uint32_t)(x >> 32) << 16 : (uint32_t)(x >> 32);
}

// launch(list) for lists that cover the k tensors in tiles of TILE elements.  With
// outputs, tensors that lie directly behind one another on both sides are one (the
// views of a flat bucket): 701 of 566 MB in all are clipped in 173 us instead of 194,
// 1200 of 8 KB in 7 instead of 17.  A norm keeps them apart: its bits depend on how
// the sum is cut, and ranks that hold the same gradients at other addresses must get
// the same norm.
template <typename T, typename O, unsigned TILE, bool OWN_OUT, typename Launch>
int for_lists(const void* const* grads, void* const* outs, const size_t* ns, int k, Launch launch) {
  constexpr size_t kMaxTiles = ((size_t)1 << (32 - log2_of(TILE))) - 1;
  List<OWN_OUT> l;
  l.k = 0;
  l.first[0] = 0;
  l.base = nullptr;
  l.out_base = nullptr;
  for (int j = 0, next; j < k; j = next) {
    size_t n = ns[j];
    for (next = j + 1; n && outs && next < k; ++next) {
      if (!ns[next]) continue;
      if ((const T*)grads[next] != (const T*)grads[j] + n || (O*)outs[next] != (O*)outs[j] + n) break;
      n += ns[next];
    }
    for (size_t at = 0; at < n;) {
      size_t tiles = l.first[l.k] >> log2_of(TILE);
      if (l.k == List<OWN_OUT>::kMost || tiles == kMaxTiles) {
        index<TILE>(l);
        if (launch(l)) return -1;
        l.k = 0;
        l.first[0] = 0;
        tiles = 0;
      }
      const size_t left = n - at, room = (kMaxTiles - tiles) * TILE, take = left < room ? left : room;
      put_address(l.lo, l.hi, l.k, (const T*)grads[j] + at);
      if constexpr (OWN_OUT) put_address(l.out_lo, l.out_hi, l.k, (const O*)outs[j] + at);
      if (!l.base) {
        l.base = (const char*)grads[j];
        l.out_base = outs ? (char*)outs[j] : nullptr;
      }
      l.first[l.k] |= (uint32_t)((take - 1) % TILE);
      l.first[++l.k] = (uint32_t)((tiles + (take + TILE - 1) / TILE) << log2_of(TILE));
      at += take;
    }
  }
  if (!l.k) return 0;
  index<TILE>(l);
  return launch(l);
}

// Whether the outputs lie to each other as the gradients do.
template <typename T, typename O>
bool same_places(void* const* outs, const void* const* grads, const size_t* ns, int k) {
  int j0 = -1;
  for (int j = 0; j < k; ++j) {
    if (!ns[j]) continue;
    if (j0 < 0) j0 = j;
    const intptr_t in = (intptr_t)grads[j] - (intptr_t)grads[j0], out = (intptr_t)outs[j] - (intptr_t)outs[j0];
    if (in / (intptr_t)sizeof(T) * (intptr_t)sizeof(O) != out) return false;
  }
  return true;
}

int finish(const char* what, const double* work, int held, double* sumsq, hipStream_t s) {
  hipLaunchKernelGGL(k_grad_finish, dim3(1), dim3(kFinishBlock), 0, s, work, held, sumsq);
  return launched(what);
}

// Up to here one block of 1024 threads does a call in one launch, without a second
// one to join the sums of several blocks.  Called one behind the other, one block or
// two launches take
//   a norm of 256 KiB             f32 5.0, 6.2 us   bf16 6.4, 6.2 us
//   a fold of 2 sources, 256 KiB      4.5, 6.0           6.9, 6.0  (4 sources 6.0, 6.0)
//   the same, 480 KiB in all          6.2, 6.1          11.0, 6.1
// as a 16-bit value takes two conversions and half the bytes.  A fold without a sum
// has none to join: 2 bf16 sources, 480 KiB in all, take many blocks 2.3 us in a graph,
// one block 10.2.  Joining the sums in the same launch, by the block that finishes last,
// loses from 128 blocks on: their counter is one address across eight dies (1024 blocks
// 37 us, two launches 10.3).
constexpr size_t kOneBlockNorm = 256u << 10;
constexpr size_t kOneBlockTile = 64u << 10;       // what it takes at a time, 4 vectors per thread
template <typename T> constexpr size_t kOneBlockFold = (sizeof(T) == 2 ? 256u : 512u) << 10;
constexpr size_t kInfinityCache = 256u << 20;

// The blocks of a norm launch: 3 of 256 threads per CU (4 for f64) lead, and leave
// few sums to join: 1.34 GB of bf16 190 us, with 2 per CU 236, with 4 196, with 8
// 221, with 32 201; 1.2 GB of f64 169 us, with 3 per CU 188, with 32 178.
template <typename T> constexpr int kBlocksPerCu = sizeof(T) == 8 ? 4 : 3;

template <typename T, int BLOCK, int UNROLL, bool NT>
int sumsq_shape(const void* const* grads, const size_t* ns, int k, double* sumsq, double* work, bool one,
                hipStream_t s) {
  constexpr unsigned kTile = BLOCK * UNROLL * kWidth<T>;
  const unsigned full = (unsigned)pgk_cu_count() * kBlocksPerCu<T>;
  const unsigned most = one ? 1 : full < (unsigned)kMaxParts ? full : kMaxParts;
  double* const parts = one ? sumsq : work;
  int held = 0;
  const int rc = for_lists<T, T, kTile, false>(grads, nullptr, ns, k, [&](const List<false>& l) {
    const unsigned tiles = tiles_of<kTile>(l), grid = tiles < most ? tiles : most;
    hipLaunchKernelGGL((k_grad_sumsq<T, BLOCK, UNROLL, NT>), dim3(grid), dim3(BLOCK), 0, s, l, grid, parts, held);
    if ((int)grid > held) held = (int)grid;
    return launched("grad_sumsq");
  });
  if (rc || (one && held)) return rc;
  return finish("grad_sumsq", work, held, sumsq, s);
}

template <typename T>
int sumsq_t(const void* const* grads, const size_t* ns, int k, double* sumsq, double* work, hipStream_t s) {
  size_t tiles = 0, bytes = 0;
  for (int j = 0; j < k; ++j) {
    tiles += (ns[j] * sizeof(T) + kOneBlockTile - 1) / kOneBlockTile;
    bytes += ns[j] * sizeof(T);
  }
  if (tiles <= kOneBlockNorm / kOneBlockTile) return sumsq_shape<T, 1024, 4, false>(grads, ns, k, sumsq, work, true, s);
  if (bytes <= kInfinityCache) return sumsq_shape<T, 256, 4, false>(grads, ns, k, sumsq, work, false, s);
  return sumsq_shape<T, 256, 4, true>(grads, ns, k, sumsq, work, false, s);
}

template <typename T, typename O, bool OWN_OUT>
int clip_lists(void* const* outs, const void* const* grads, const size_t* ns, int k, const double* sumsq, int nsum,
               double scale, double max_norm, double* norm, hipStream_t s) {
  constexpr unsigned kTile = kClipTile<T, O>;
  bool any = false;
  auto launch = [&](const List<OWN_OUT>& l) {
    hipLaunchKernelGGL((k_grad_clip<T, O, OWN_OUT>), dim3(tiles_of<kTile>(l)), dim3(kClipBlock), 0, s, l, sumsq, nsum,
                       scale, max_norm, any ? nullptr : norm);
    any = true;
    return launched("grad_clip");
  };
  const int rc = for_lists<T, O, kTile, OWN_OUT>(grads, outs, ns, k, launch);
  if (rc || any || !norm) return rc;
  hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(64), 0, s, sumsq, nsum, scale, norm);
  return launched("grad_clip");
}

template <typename T, typename O>
int clip_t(void* const* outs, const void* const* grads, const size_t* ns, int k, const double* sumsq, int nsum,
           double scale, double max_norm, double* norm, hipStream_t s) {
  return same_places<T, O>(outs, grads, ns, k)
             ? clip_lists<T, O, false>(outs, grads, ns, k, sumsq, nsum, scale, max_norm, norm, s)
             : clip_lists<T, O, true>(outs, grads, ns, k, sumsq, nsum, scale, max_norm, norm, s);
}

template <typename T, int NS>
void burst_launch(T* out, const Sources& src, size_t e0, size_t e1, double scale, double* parts, int held,
                  unsigned grid, int tiles, hipStream_t s) {
  if (tiles == 32)
    hipLaunchKernelGGL((k_grad_fold_burst<T, NS, 32>), dim3(grid), dim3(kBurstBlock), 0, s, out, src, e0, e1, scale,
                       parts, held);
  else
    hipLaunchKernelGGL((k_grad_fold_burst<T, NS, 16>), dim3(grid), dim3(kBurstBlock), 0, s, out, src, e0, e1, scale,
                       parts, held);
}

template <typename T, typename O>
int fold_t(void* out, const Sources& src, int nsrc, size_t n, double scale, double* sumsq, double* work,
           hipStream_t s) {
  O* o = (O*)out;
  const bool one = sumsq && n * (nsrc * sizeof(T) + sizeof(O)) <= kOneBlockFold<T>;
  double* parts = !sumsq ? nullptr : one && n ? sumsq : work;
  size_t e0 = 0;
  int held = 0;
  auto ran = [&](unsigned grid, size_t e1) {
    if ((int)grid > held) held = (int)grid;
    e0 = e1;
    return launched("grad_fold");
  };
  // the launches of the burst form hold what the waves' registers hold: 512 blocks (two per CU) of 32
  // vectors per thread, then one of 512 to 1024 blocks of 16; what is left, under 32 MiB per source,
  // goes a vector per thread
  if constexpr (std::is_same_v<T, O>) {
    constexpr size_t kHalf = (size_t)512 * kBurstBlock * 16 * kWidth<T>;      // 32 MiB per source
    while (nsrc >= 5 && nsrc <= 8 && n - e0 >= kHalf) {
      const int tiles = n - e0 >= 2 * kHalf ? 32 : 16;
      const size_t per = (size_t)kBurstBlock * tiles * kWidth<T>;
      const size_t take = tiles == 32 ? 2 * kHalf : (n - e0) / kWidth<T> * kWidth<T>;
      const unsigned grid = (unsigned)((take + per - 1) / per);
      switch (nsrc) {
        case 5: burst_launch<T, 5>(o, src, e0, e0 + take, scale, parts, held, grid, tiles, s); break;
        case 6: burst_launch<T, 6>(o, src, e0, e0 + take, scale, parts, held, grid, tiles, s); break;
        case 7: burst_launch<T, 7>(o, src, e0, e0 + take, scale, parts, held, grid, tiles, s); break;
        default: burst_launch<T, 8>(o, src, e0, e0 + take, scale, parts, held, grid, tiles, s);
      }
      if (ran(grid, e0 + take)) return -1;
    }
  }
  if (e0 < n) {
    constexpr size_t per = (size_t)kFoldBlock * kWidth<O>;
    const size_t tiles = (n - e0 + per - 1) / per;
    const unsigned grid = one ? 1 : tiles < (size_t)kMaxParts ? (unsigned)tiles : kMaxParts;
    switch (nsrc) {
#define PGK_FOLD_CASE(NS, K) \
      K: hipLaunchKernelGGL((k_grad_fold<T, O, NS>), dim3(grid), dim3(kFoldBlock), 0, s, o, src, nsrc, e0, n, scale, \
                            parts, held); break;
      PGK_FOLD_CASE(1, case 1) PGK_FOLD_CASE(2, case 2) PGK_FOLD_CASE(3, case 3) PGK_FOLD_CASE(4, case 4)
      PGK_FOLD_CASE(5, case 5) PGK_FOLD_CASE(6, case 6) PGK_FOLD_CASE(7, case 7) PGK_FOLD_CASE(kMaxUnrolled, default)
#undef PGK_FOLD_CASE
    }
    if (ran(grid, n)) return -1;
  }
  return parts && parts != sumsq ? finish("grad_fold", work, held, sumsq, s) : 0;
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
      !check_work(what, sumsq, work) || !check_apart(what, "sumsq", sumsq, 8, grads, ns, k, elem_size(dt)) ||
      !check_apart(what, "work", work, PGK_GRAD_WORK_BYTES, grads, ns, k, elem_size(dt))) return -1;
  return with_types(dt, dt, [&](auto* t, auto*) {
    return sumsq_t<std::remove_pointer_t<decltype(t)>>(grads, ns, k, sumsq, (double*)work, (hipStream_t)stream);
  });
}

int pgk_grad_clip_check(void* const* outs, int out_dt, const void* const* grads, int dt, const size_t* ns, int k,
                        double scale, double max_norm) {
  const char* what = "grad_clip";
  if (!check_types(what, dt, out_dt) || !check_list(what, grads, ns, k, elem_size(dt)) ||
      !check_list(what, (const void* const*)outs, ns, k, elem_size(out_dt))) return -1;
  if (!isfinite(scale)) { set_err("pgk: %s: scale %g", what, scale); return -1; }
  if (!(max_norm >= 0)) { set_err("pgk: %s: max_norm %g", what, max_norm); return -1; }
  for (int j = 0; j < k; ++j)
    if (ns[j] && !(outs[j] == grads[j] && dt == out_dt) &&
        overlap(outs[j], ns[j] * elem_size(out_dt), grads[j], ns[j] * elem_size(dt))) {
      set_err("pgk: %s: output %d overlaps its gradient at a different address", what, j);
      return -1;
    }
  return 0;
}

int pgk_grad_clip(void* const* outs, int out_dt, const void* const* grads, int dt, const size_t* ns, int k,
                  const double* sumsq, int nsum, double scale, double max_norm, double* norm, void* stream) {
  const char* what = "grad_clip";
  if (pgk_grad_clip_check(outs, out_dt, grads, dt, ns, k, scale, max_norm) || !check_sums(what, sumsq, "sumsq") ||
      (norm && !check_sums(what, norm, "norm"))) return -1;
  if (nsum < 1) { set_err("pgk: %s: %d partial sums", what, nsum); return -1; }
  if (norm && overlap(norm, 8, sumsq, (size_t)nsum * 8)) { set_err("pgk: %s: norm lies in sumsq", what); return -1; }
  const void* const* const o = (const void* const*)outs;
  if (!check_apart(what, "sumsq", sumsq, (size_t)nsum * 8, o, ns, k, elem_size(out_dt)) ||
      (norm && (!check_apart(what, "norm", norm, 8, o, ns, k, elem_size(out_dt)) ||
                !check_apart(what, "norm", norm, 8, grads, ns, k, elem_size(dt))))) return -1;
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
  if (sumsq && !check_work(what, sumsq, work)) return -1;
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
    if (sumsq && (!check_apart(what, "sumsq", sumsq, 8, o, same, 1, oes) ||
                  !check_apart(what, "sumsq", sumsq, 8, srcs, same, nsrc, es) ||
                  !check_apart(what, "work", work, PGK_GRAD_WORK_BYTES, o, same, 1, oes) ||
                  !check_apart(what, "work", work, PGK_GRAD_WORK_BYTES, srcs, same, nsrc, es))) return -1;
  } else if (!sumsq) {
    return 0;
  }
  return with_types(dt, out_dt, [&](auto* t, auto* o) {
    return fold_t<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>>(
        out, src, nsrc, n, scale, sumsq, (double*)work, (hipStream_t)stream);
  });
}

}  // extern "C"
