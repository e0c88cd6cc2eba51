// The end of a training step on gfx950: the global 2-norm of many gradient tensors, and the AdamW
// step over many parameter tensors with its two states in fp32 or in 8 bits.
//
// All of it is bound by HBM: every gradient, parameter and state is read once and written once.
// Tensors travel in kernel arguments (4 KB of pointers and sizes at most), so nothing is copied to
// the device and a call can be captured.  The norm reads them there (228 gradients a launch); the
// step's first kernels, one for every 99 tensors with fp32 states or 70 with 8-bit ones, write
// them to a table in the workspace, and one launch then runs over all tensors: with a launch for
// every 63 tensors the step of 392 adapters with 8-bit states took 138 us, 8 us of each launch its
// beginning and end.
//
// 8-bit states: blocks of 256 values in storage order share one fp32 scale, the largest magnitude;
// a value is kept as the code of the nearest of 256 book values times that scale.  The update
// and the choice of the code are computed in fp64: a value next to the border of two codes
// takes the side that the exact recurrence says (in fp32 one value in 10^5 took the other one,
// one whole code off), and the fp64 units have the time, since the pass waits for HBM.
#include "common.h"
#include "mxs_nf4.h"

namespace mxs {

typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef double double2_t __attribute__((ext_vector_type(2)));

constexpr int kStateBlock = 256;  // 8-bit values per scale
constexpr int kTableArgs = 3960;  // bytes of tensors in a launch's arguments

// ---- code books -------------------------------------------------------------------------------

// The 8-bit dynamic map (Dettmers, arXiv 1511.04561), ascending: the signed one is the code book
// of the nested absmax; the unsigned one has a bit more of fraction (2^(i+1) midpoints in decade
// i instead of 2^i and their negatives).  Both hold 0 and 1.
//
// The nearest code of x, relative to its block's largest magnitude, is the number of borders
// (midpoints of neighbours) below it.  The leading 16 bits of |x| plus an offset pick an interval
// that holds one border at most, and whose ends no border comes near (within 2^-14, relative: many
// borders lie on fractions of few bits, where the intervals would end without the offset): the
// code is the count of borders below the interval, and one more if its border is below x.  In
// fp32 that is sure unless x is within 2^-20 of the border, relative; then, one value in 10^4 or
// so, it is decided in fp64, where border times scale is exact.
constexpr uint32_t kKeyOffset = 0xa8f0;
constexpr int kKeyBase = (0x34000000 + kKeyOffset) >> 16;  // of 2^-23: no border is nearer to 0
constexpr int kKeys = ((0x3f800000 + kKeyOffset) >> 16) - kKeyBase + 1;  // up to 1

constexpr float key_end(int k) {  // where interval k begins
  return __builtin_bit_cast(float, ((uint32_t)(kKeyBase + k) << 16) - kKeyOffset);
}

struct Book {
  double value[256];
  float border[256];  // border[c]: a value above it is nearer to code c + 1; [255] is infinite
  uint8_t below[2 * kKeys + 2];  // borders below the interval of |x|, and of -|x| from kKeys on
};

struct Border64 {
  double at[256];
};

constexpr Book make_book(bool is_signed) {
  Book b{};
  constexpr double decade[7] = {1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 1e-1, 1.0};
  int at = is_signed ? 127 : 0;  // index of zero
  const int zero = at;
  b.value[at++] = 0.0;
  for (int i = 0; i < 7; i++) {
    const int n = is_signed ? 1 << i : 2 << i;
    for (int j = 0; j < n; j++) {
      const float lo = (float)(0.1 + 0.9 * j / n), hi = (float)(0.1 + 0.9 * (j + 1) / n);
      const float mid = (lo + hi) / 2.0f;
      const float v = (float)(decade[i] * (double)mid);
      if (is_signed) b.value[2 * zero - at] = -v;
      b.value[at++] = v;
    }
  }
  b.value[255] = 1.0;
  for (int c = 0; c < 255; c++) b.border[c] = (float)((b.value[c] + b.value[c + 1]) / 2);
  b.border[255] = __builtin_huge_valf();
  int c = 0;
  for (int k = 0; k < kKeys; k++) {
    while (k > 0 && c < 255 && b.border[c] < key_end(k)) c++;
    if (k == 0) c = zero;  // borders below 0
    b.below[k] = (uint8_t)c;
    int d = zero;
    while (d > 0 && b.border[d - 1] >= -key_end(k + 1)) d--;
    b.below[kKeys + k] = (uint8_t)d;
  }
  return b;
}

constexpr Border64 make_borders(const Book& b) {
  Border64 r{};
  for (int c = 0; c < 255; c++) r.at[c] = (b.value[c] + b.value[c + 1]) / 2;  // 25 bits: exact
  r.at[255] = __builtin_huge_val();
  return r;
}

// One border at most in an interval of either sign, and none within 2^-14 of its ends, relative.
constexpr bool book_ok(const Book& b, int zero) {
  for (int side = 0; side < 2; side++) {
    int c = side ? zero - 1 : zero;  // outwards from 0
    for (int k = 0; k < kKeys; k++) {
      int in = 0;
      const double lo = key_end(k), hi = key_end(k + 1);
      for (; c >= 0 && c < 255; c += side ? -1 : 1) {
        const double a = side ? -b.border[c] : b.border[c];
        if (a > hi * (1 - 0x1p-14) && a < hi * (1 + 0x1p-14)) return false;
        if (a < lo || a >= hi) break;
        in++;
      }
      if (in > 1) return false;
    }
    if (c >= 0 && c < 255) return false;
  }
  return true;
}

constexpr Book kSignedBook = make_book(true), kUnsignedBook = make_book(false);
static_assert(book_ok(kSignedBook, 127) && book_ok(kUnsignedBook, 0), "intervals of the search");
__device__ __constant__ static const Book kBooks[2] = {kSignedBook, kUnsignedBook};
__device__ __constant__ static const Border64 kBorders[2] = {make_borders(kSignedBook),
                                                             make_borders(kUnsignedBook)};

// The code whose value times `top` is nearest to x (the lower one of two as near); xf is x rounded
// to fp32, inv 1 / top within two roundings (0 for a block of zeros).
template <bool SIGNED>
__device__ __forceinline__ int nearest_code(const Book& b, double x, float xf, float top,
                                            float inv) {
  const float f = xf * inv;
  int k = (int)(((__builtin_bit_cast(uint32_t, f) & 0x7fffffffu) + kKeyOffset) >> 16) - kKeyBase;
  k = min(max(k, 0), kKeys - 1);
  if (SIGNED && f < 0.0f) k += kKeys;
  const int c = b.below[k];
  const float at = b.border[c];
  bool above = at < f;
  if (fabsf(f - at) <= fabsf(at) * 0x1p-20f)
    above = kBorders[SIGNED ? 0 : 1].at[c] * (double)top < x;
  return c + (above ? 1 : 0);
}

// ---- element access ---------------------------------------------------------------------------

// Eight values from index i of n (zeros past the end).  vec: the pointer is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t i, int64_t n, bool vec, float (&x)[8]) {
  typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int W = 16 / sizeof(T);
  if (vec && i + 8 <= n) {
#pragma unroll
    for (int q = 0; q < 8 / W; q++) {
      const vec_t v = *reinterpret_cast<const vec_t*>(p + i + q * W);
#pragma unroll
      for (int e = 0; e < W; e++) x[q * W + e] = (float)v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = i + e < n ? (float)p[i + e] : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t i, int64_t n, bool vec, const float (&x)[8]) {
  typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int W = 16 / sizeof(T);
  if (vec && i + 8 <= n) {
#pragma unroll
    for (int q = 0; q < 8 / W; q++) {
      vec_t v;
#pragma unroll
      for (int e = 0; e < W; e++) v[e] = (T)x[q * W + e];
      *reinterpret_cast<vec_t*>(p + i + q * W) = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (i + e < n) p[i + e] = (T)x[e];
  }
}

__device__ __forceinline__ void load8_codes(const uint8_t* p, int64_t i, int64_t n, bool vec,
                                            int (&c)[8]) {
  if (vec && i + 8 <= n) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p + i);
#pragma unroll
    for (int e = 0; e < 8; e++) c[e] = (v[e >> 2] >> (8 * (e & 3))) & 255;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) c[e] = i + e < n ? p[i + e] : 0;
  }
}

__device__ __forceinline__ void store8_codes(uint8_t* p, int64_t i, int64_t n, bool vec,
                                             const int (&c)[8]) {
  if (vec && i + 8 <= n) {
    u32x2 v = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++) v[e >> 2] |= (uint32_t)c[e] << (8 * (e & 3));
    *reinterpret_cast<u32x2*>(p + i) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (i + e < n) p[i + e] = (uint8_t)c[e];
  }
}

// ---- tables -----------------------------------------------------------------------------------

// A tensor of a step, or 2^31 values of one: chunks [start, next entry's start).
constexpr uint32_t kVecBit = 0x80000000u;  // of `start`: the pointers are 16-byte aligned

struct StepTensor {
  void* p;
  const void* g;
  void *m, *v;
  uint32_t n, start;
};
struct StepTensor8 {
  void* p;
  const void* g;
  void *m, *v;
  float *ms, *vs;
  uint32_t n, start;
};

template <typename E>
struct StepPart {  // entries of one set-up launch
  static constexpr int N = kTableArgs / sizeof(E);
  E t[N];
};

constexpr int kVec = 16;  // of the norm's flags, beside MXS_DTYPE_*
// Gradients of one launch of the norm; a longer one than 2^31 values takes several entries.
struct NormTable {
  static constexpr int N = (kTableArgs - 8) / 17;
  const void* g[N];
  uint32_t n[N];
  int start[N + 1];
  uint8_t flags[N];
  int count;
};

// The tensor of chunk `c` (uniform).
template <typename Tab>
__device__ __forceinline__ int tensor_of(const Tab& tab, int c) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c >= tab.start[mid]) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The entry of chunk `c` (uniform) of a step's table: halved down to 256 entries, which the lanes
// look through together.
template <typename E>
__device__ __forceinline__ int entry_of(const E* tab, int count, uint32_t c) {
  int lo = 0, hi = count;
  while (hi - lo > 256) {
    const int mid = (lo + hi) >> 1;
    if (c >= (tab[mid].start & ~kVecBit)) lo = mid;
    else hi = mid;
  }
  int n = 0;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int i = lo + 64 * j + lane;
    n += __popcll(__ballot(i < hi && (tab[i < hi ? i : lo].start & ~kVecBit) <= c));
  }
  return __builtin_amdgcn_readfirstlane(lo + n - 1);
}

// ---- gradient norm ----------------------------------------------------------------------------

constexpr int kNormChunk = 8192;  // values of a workgroup

// Sum of 256 lanes' values in a fixed order; the result in lane 0.
__device__ __forceinline__ double sum256(double x, double* s) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  return s[0] + s[1] + s[2] + s[3];
}

template <typename T>
__device__ __forceinline__ double squares(const T* g, int64_t i0, int64_t n, bool vec) {
  double a[2] = {0.0, 0.0};
#pragma unroll
  for (int u = 0; u < kNormChunk / 2048; u++) {
    float x[8];
    load8(g, i0 + u * 2048 + threadIdx.x * 8, n, vec, x);
#pragma unroll
    for (int e = 0; e < 8; e++) a[e & 1] += (double)x[e] * (double)x[e];
  }
  return a[0] + a[1];
}

constexpr int kNormGroups = 16384;  // workgroups of a launch at most

// Sums of squares per workgroup, in fp64: the squares of any fp32 and their sums are then neither
// infinite nor lost, whatever their sizes.
__global__ __launch_bounds__(256) void k_norm_chunks(NormTable tab, double* partial) {
  __shared__ double s[4];
  double a = 0.0;
  for (int c = (int)blockIdx.x; c < tab.start[tab.count]; c += (int)gridDim.x) {
    const int i = tensor_of(tab, c);
    const int64_t at = (int64_t)(c - tab.start[i]) * kNormChunk, n = tab.n[i];
    const bool vec = tab.flags[i] & kVec;
    switch (tab.flags[i] & (kVec - 1)) {
      case MXS_DTYPE_F16: a += squares(static_cast<const _Float16*>(tab.g[i]), at, n, vec); break;
      case MXS_DTYPE_BF16: a += squares(static_cast<const __bf16*>(tab.g[i]), at, n, vec); break;
      default: a += squares(static_cast<const float*>(tab.g[i]), at, n, vec);
    }
  }
  a = sum256(a, s);
  if (threadIdx.x == 0) partial[blockIdx.x] = a;
}

__global__ __launch_bounds__(1024) void k_norm_finish(const double* partial, int64_t n,
                                                      const float* grad_scale, float* out) {
  __shared__ double s[16];
  double a = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) a += partial[i];
#pragma unroll
  for (int o = 32; o; o >>= 1) a += __shfl_xor(a, o);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x) return;
  a = 0.0;
  for (int w = 0; w < 16; w++) a += s[w];
  out[0] = (float)(sqrt(a) / (grad_scale ? (double)grad_scale[0] : 1.0));
}

// ---- AdamW ------------------------------------------------------------------------------------

// What every value of a step shares, computed once per call.
struct StepScalars {
  double coef;    // gradients times this: clipping and the loss scale
  float keep;     // 1 - lr * weight_decay
  float size;     // lr / (1 - beta1^t)
  float root;     // 1 / sqrt(1 - beta2^t)
  int skip;       // an overflow was found: nothing is changed
};

struct StepInputs {
  float* step;
  double lr;
  const float* lr_dev;
  double beta1, beta2, weight_decay;
  const float* norm;
  double max_norm;
  const float *grad_scale, *found_inf;
};

// Entries of the table from kernel arguments to memory; the first launch of a step also computes
// what its values share.
template <typename E>
__global__ __launch_bounds__(256) void k_adamw_setup(StepPart<E> part, int count, E* table,
                                                     StepScalars* out, StepInputs in) {
  const uint32_t* src = reinterpret_cast<const uint32_t*>(part.t);
  uint32_t* dst = reinterpret_cast<uint32_t*>(table);
  for (int i = threadIdx.x; i < count * (int)(sizeof(E) / 4); i += 256) dst[i] = src[i];
  if (!out || threadIdx.x) return;
  const int skip = in.found_inf && in.found_inf[0] != 0.0f;
  const float t = in.step[0] + 1.0f;
  const double lr = in.lr_dev ? (double)in.lr_dev[0] : in.lr;
  double coef = 1.0;
  if (in.norm) {
    coef = in.max_norm / ((double)in.norm[0] + 1e-6);
    if (coef > 1.0) coef = 1.0;  // a NaN stays one
  }
  if (in.grad_scale) coef /= (double)in.grad_scale[0];
  out->coef = coef;
  out->keep = (float)(1.0 - lr * in.weight_decay);
  out->size = (float)(lr / (1.0 - pow(in.beta1, (double)t)));
  out->root = (float)(1.0 / sqrt(1.0 - pow(in.beta2, (double)t)));
  out->skip = skip;
  if (!skip) in.step[0] = t;
}

// m / (sqrt(v) root + eps) with the hardware's root and reciprocal, each within one step of fp32;
// roots of values below 2^-96 are taken 2^48 times larger.
__device__ __forceinline__ float ratio(float m, float v, float root, float eps) {
  const bool low = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(low ? v * 0x1p96f : v) * (low ? 0x1p-48f : 1.0f);
  return m * __builtin_amdgcn_rcpf(r * root + eps);
}

constexpr int kStepChunk = 2048;  // values of a workgroup, fp32 states

template <typename T>
__device__ __forceinline__ void step32(const StepTensor& t, int64_t i, bool vec,
                                       const StepScalars& s, float b1, float b2, float c1,
                                       float c2, float eps) {
  float p[8], g[8], m[8], v[8];
  T* tp = static_cast<T*>(t.p);
  float *tm = static_cast<float*>(t.m), *tv = static_cast<float*>(t.v);
  load8(static_cast<const T*>(t.g), i, t.n, vec, g);
  load8(tm, i, t.n, vec, m);
  load8(tv, i, t.n, vec, v);
  load8(tp, i, t.n, vec, p);
  const float coef = (float)s.coef;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float x = g[e] * coef;
    m[e] = b1 * m[e] + c1 * x;
    v[e] = b2 * v[e] + c2 * (x * x);
    p[e] = p[e] * s.keep - s.size * ratio(m[e], v[e], s.root, eps);
  }
  store8(tm, i, t.n, vec, m);
  store8(tv, i, t.n, vec, v);
  store8(tp, i, t.n, vec, p);
}

// fp32 states, one pass: 28 bytes a value with fp32 parameters, 22 with 16-bit ones.
template <typename T>
__global__ __launch_bounds__(256) void k_adamw(const StepTensor* __restrict__ tab, int count,
                                               const StepScalars* scalars, float b1, float b2,
                                               float c1, float c2, float eps) {
  const StepScalars s = *scalars;
  if (s.skip) return;
  const StepTensor& t = tab[entry_of(tab, count, blockIdx.x)];
  const int64_t at =
      (int64_t)(blockIdx.x - (t.start & ~kVecBit)) * kStepChunk + threadIdx.x * 8;
  if (at < t.n) step32<T>(t, at, (t.start & kVecBit) != 0, s, b1, b2, c1, c2, eps);
}

constexpr uint32_t kStep8Groups = 2048;  // workgroups at most (1024 and 4096: within 1 %, 2 % more)
constexpr int kStep8Chunk = 2048;  // values of a workgroup, 8-bit states: 8 blocks

// The largest of 32 lanes' magnitudes (a block of 256 values lies in half a wave), as bits: those
// of a NaN are above all others.
__device__ __forceinline__ uint32_t max32(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 15, 15, true));   // lane ^ 1
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 15, 15, true));   // lane ^ 2
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 15, 15, true));  // 7 - lane
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 15, 15, true));  // 15 - lane
  return max(x, (uint32_t)__shfl_xor((int)x, 16));
}

// New values x[8] of a block as codes and the block's scale.  A block with a value that is not
// finite gets a NaN scale: all of its values are then NaN, as they are lost.
template <bool SIGNED>
__device__ __forceinline__ float encode(const Book& b, const double (&x)[8], int (&c)[8]) {
  float f[8];
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    f[e] = (float)x[e];
    bits = max(bits, __builtin_bit_cast(uint32_t, f[e]) & 0x7fffffffu);
  }
  bits = max32(bits);
  float top = __builtin_bit_cast(float, bits);
  if (bits >= 0x7f800000u) top = __builtin_nanf("");
  // A scale below fp32's normal range has no fp32 reciprocal: both sides times 2^64 then.
  const bool low = top < 0x1p-100f;
  const float up = low ? 0x1p64f : 1.0f;
  const float inv = top > 0.0f ? __builtin_amdgcn_rcpf(top * up) : 0.0f;
  if (__any(low)) {  // (rare: kept apart, so that its products are not always paid for)
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] *= up;
  }
#pragma unroll
  for (int e = 0; e < 8; e++) c[e] = nearest_code<SIGNED>(b, x[e], f[e], top, inv);
  return top;
}

// Eight values of a step as they are loaded.
template <typename T>
struct Raw8 {
  static constexpr int W = sizeof(T) / 2;
  u32x4 p[W], g[W];
  u32x2 m, v;
  float sm, sv;
};

template <typename T>
__device__ __forceinline__ void widen(const u32x4 (&x)[sizeof(T) / 2], float (&f)[8]) {
  typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int W = 16 / sizeof(T);
#pragma unroll
  for (int q = 0; q < 8 / W; q++) {
    const vec_t v = __builtin_bit_cast(vec_t, x[q]);
#pragma unroll
    for (int e = 0; e < W; e++) f[q * W + e] = (float)v[e];
  }
}

// The step of eight values; `in` says which of them exist (ALL: every one).
template <bool ALL>
__device__ __forceinline__ void step8(float (&p)[8], const float (&g)[8], int (&cm)[8],
                                      int (&cv)[8], float& sm, float& sv, int in,
                                      const StepScalars& s, const Book* books, double b1,
                                      double b2, float eps) {
  // Products and sums rounded one by one: (9 x + y) / 10 of numbers as short as these can lie
  // half way between two fp32 scales, where a fused sum would decide otherwise than the formula.
#pragma clang fp contract(off)
  const double d1 = 1.0 - b1, d2 = 1.0 - b2, sm64 = (double)sm, sv64 = (double)sv;
  double m[8], v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const double x = (double)g[e] * s.coef;
    const bool live = ALL || e < in;
    m[e] = live ? books[0].value[cm[e]] * sm64 * b1 + x * d1 : 0.0;
    v[e] = live ? books[1].value[cv[e]] * sv64 * b2 + (x * x) * d2 : 0.0;
    p[e] = p[e] * s.keep - s.size * ratio((float)m[e], (float)v[e], s.root, eps);
  }
  sm = encode<true>(books[0], m, cm);
  sv = encode<false>(books[1], v, cv);
}

__device__ __forceinline__ void books_to_lds(Book* books) {
  const uint32_t* src = reinterpret_cast<const uint32_t*>(kBooks);
  uint32_t* dst = reinterpret_cast<uint32_t*>(books);
  for (int i = threadIdx.x; i < (int)(2 * sizeof(Book) / 4); i += blockDim.x) dst[i] = src[i];
  __syncthreads();
}

// 8-bit states, one pass: 10 bytes a value with 16-bit parameters, 16 with fp32 ones.  A wave takes
// 512 values, two blocks.  About 70 vector instructions a value fill the pass as much as its bytes
// do: 323 M bf16 values take 959 us, 3.4 TB/s.  Loading ahead of the values in hand cost more
// registers, and so waves, than it gained (1121 us); the entry read anew for every chunk, behind
// stores that might have changed it, 1130 us.
template <typename T>
__global__ __launch_bounds__(256, 4) void k_adamw8(const StepTensor8* __restrict__ tab, int count,
                                                   uint32_t chunks,
                                                const StepScalars* scalars, double b1, double b2,
                                                float eps) {
  __shared__ Book books[2];
  const StepScalars s = *scalars;
  if (s.skip) return;
  uint32_t start = 0, end = 0;  // chunks of the entry in hand; most steps to the next stay in it
  StepTensor8 t = {};
  int64_t at = 0;      // the lane's first value
  bool whole = false;  // the wave's 512 values exist and are aligned
  auto place = [&](uint32_t c) {
    if (c >= end) {
      const int i = entry_of(tab, count, c);
      t = tab[i];
      start = t.start & ~kVecBit;
      end = i + 1 < count ? tab[i + 1].start & ~kVecBit : chunks;
    }
    at = (int64_t)(c - start) * kStep8Chunk + threadIdx.x * 8;
    whole = (t.start & kVecBit) && at - threadIdx.x % 64 * 8 + 512 <= t.n;
  };
  auto load = [&](Raw8<T>& r) {
    if (!whole) return;
    const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const T*>(t.p) + at);
    const u32x4* g = reinterpret_cast<const u32x4*>(static_cast<const T*>(t.g) + at);
#pragma unroll
    for (int q = 0; q < Raw8<T>::W; q++) r.g[q] = g[q], r.p[q] = p[q];
    r.m = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(t.m) + at);
    r.v = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(t.v) + at);
    r.sm = t.ms[at / kStateBlock];
    r.sv = t.vs[at / kStateBlock];
  };
  Raw8<T> raw;
  place(blockIdx.x);
  load(raw);  // on its way while the books come
  books_to_lds(books);
  for (uint32_t c = blockIdx.x;;) {
    T* tp = static_cast<T*>(t.p);
    uint8_t *tm = static_cast<uint8_t*>(t.m), *tv = static_cast<uint8_t*>(t.v);
    const int64_t i = at, n = t.n, blk = i / kStateBlock;
    float p[8], g[8], sm, sv;
    int cm[8], cv[8];
    if (whole) {
      widen<T>(raw.p, p);
      widen<T>(raw.g, g);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        cm[e] = (raw.m[e >> 2] >> (8 * (e & 3))) & 255;
        cv[e] = (raw.v[e >> 2] >> (8 * (e & 3))) & 255;
      }
      sm = raw.sm, sv = raw.sv;
      step8<true>(p, g, cm, cv, sm, sv, 8, s, books, b1, b2, eps);
      store8(tp, i, i + 8, true, p);
      store8_codes(tm, i, i + 8, true, cm);
      store8_codes(tv, i, i + 8, true, cv);
    } else {
      const bool any = blk * kStateBlock < n;
      load8(static_cast<const T*>(t.g), i, n, false, g);
      load8_codes(tm, i, n, false, cm);
      load8_codes(tv, i, n, false, cv);
      load8(tp, i, n, false, p);
      sm = any ? t.ms[blk] : 0.0f, sv = any ? t.vs[blk] : 0.0f;
      const int in = (int)(n - i < 0 ? 0 : n - i < 8 ? n - i : 8);
      step8<false>(p, g, cm, cv, sm, sv, in, s, books, b1, b2, eps);
      store8(tp, i, n, false, p);
      store8_codes(tm, i, n, false, cm);
      store8_codes(tv, i, n, false, cv);
    }
    if ((threadIdx.x & 31) == 0 && blk * kStateBlock < n) {
      t.ms[blk] = sm;
      t.vs[blk] = sv;
    }
    c += gridDim.x;
    if (c >= chunks) break;
    place(c);
    load(raw);
  }
}

// The values that codes stand for: book value times scale, rounded once.  Four values a lane, so
// that a wave's store is 1 KB in one piece; nothing is read again, so loads and stores pass the
// caches by.
__global__ __launch_bounds__(256) void k_state_values(const uint8_t* codes, const float* scale,
                                                      float* out, int64_t n, int book, int vec) {
  __shared__ float value[256];
  value[threadIdx.x] = (float)kBooks[book].value[threadIdx.x];
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * 4096 + threadIdx.x * 4;
  if (vec && i0 - threadIdx.x * 4 + 4096 <= n) {
    uint32_t c[4];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      c[u] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(codes + i0 + u * 1024));
      s[u] = scale[(i0 + u * 1024) / kStateBlock];
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      float4_t x;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = value[(c[u] >> (8 * e)) & 255] * s[u];
      __builtin_nontemporal_store(x, reinterpret_cast<float4_t*>(out + i0 + u * 1024));
    }
  } else {
    for (int u = 0; u < 4; u++)
      for (int e = 0; e < 4; e++) {
        const int64_t i = i0 + u * 1024 + e;
        if (i < n) out[i] = value[codes[i]] * scale[i / kStateBlock];
      }
  }
}

// ---- host side --------------------------------------------------------------------------------

static bool on16(const void* p) { return ((uintptr_t)p % 16) == 0; }

static bool dtype_ok(int d) {
  return d == MXS_DTYPE_F16 || d == MXS_DTYPE_F32 || d == MXS_DTYPE_BF16;
}

static int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MXS_OK : (int)e;
}

// One step over tensors whose parameters are T: the table's entries, then the launch over them.
// `table` has room for the entries; main(table, entries, chunks) launches.
constexpr int64_t kEntryValues = (int64_t)1 << 31;  // of one entry

static int64_t step_entries(int count, const int64_t* sizes) {
  int64_t n = 0;
  for (int i = 0; i < count; i++) n += (sizes[i] + kEntryValues - 1) / kEntryValues;
  return n;
}

template <typename E, typename Fill, typename Main>
static int run_step(int count, const int64_t* sizes, const int* dtypes, int dtype, int64_t chunk,
                    E* table, StepScalars* scalars, bool& first, const StepInputs& in,
                    hipStream_t stream, Fill fill, Main main) {
  StepPart<E> part;
  int held = 0, entries = 0;
  int64_t chunks = 0;
  auto flush = [&]() {
    if (held == 0) return MXS_OK;
    hipLaunchKernelGGL(k_adamw_setup<E>, dim3(1), dim3(256), 0, stream, part, held,
                       table + entries, first ? scalars : nullptr, in);
    first = false;
    entries += held;
    held = 0;
    return launched();
  };
  for (int i = 0; i < count; i++) {
    if (dtypes[i] != dtype) continue;
    for (int64_t at = 0; at < sizes[i]; at += kEntryValues) {
      const int64_t n = sizes[i] - at < kEntryValues ? sizes[i] - at : kEntryValues;
      if (held == StepPart<E>::N) {
        const int rc = flush();
        if (rc != MXS_OK) return rc;
      }
      const bool vec = fill(part.t[held], i, at);
      part.t[held].n = (uint32_t)n;
      part.t[held].start = (uint32_t)chunks | (vec ? kVecBit : 0u);
      chunks += (n + chunk - 1) / chunk;
      if (chunks >= 1 << 24) return MXS_ERR_SIZE;  // a launch has fewer than 2^32 lanes
      held++;
    }
  }
  const int rc = flush();
  if (rc != MXS_OK || entries == 0) return rc;
  main(table, entries, (uint32_t)chunks);
  return launched();
}

static int64_t norm_chunks(int count, const int64_t* sizes) {
  int64_t n = 0;
  for (int i = 0; i < count; i++) n += (sizes[i] + kNormChunk - 1) / kNormChunk;
  return n;
}

}  // namespace mxs

using namespace mxs;

extern "C" {

int64_t mxs_grad_norm_workspace_bytes(int count, const int64_t* sizes) {
  if (count < 0 || (count && !sizes)) return MXS_ERR_ARG;
  for (int i = 0; i < count; i++)
    if (sizes[i] < 0) return MXS_ERR_ARG;
  return 8 * norm_chunks(count, sizes) + 16;
}

int mxs_grad_norm(int count, const void* const* grads, const int64_t* sizes, const int* dtypes,
                  const float* grad_scale, float* out, void* workspace, hipStream_t stream) {
  if (count < 0 || !out || !workspace || (count && (!grads || !sizes || !dtypes)))
    return MXS_ERR_ARG;
  for (int i = 0; i < count; i++) {
    if (sizes[i] < 0 || (sizes[i] && !grads[i])) return MXS_ERR_ARG;
    if (!dtype_ok(dtypes[i])) return MXS_ERR_DTYPE;
  }
  double* partial = static_cast<double*>(workspace);
  if ((uintptr_t)workspace % 8) return MXS_ERR_ALIGN;
  NormTable tab;
  int64_t groups = 0;
  tab.count = 0, tab.start[0] = 0;
  auto flush = [&]() {
    const int chunks = tab.start[tab.count], grid = chunks < kNormGroups ? chunks : kNormGroups;
    if (grid == 0) return MXS_OK;
    hipLaunchKernelGGL(k_norm_chunks, dim3(grid), dim3(256), 0, stream, tab, partial + groups);
    groups += grid;
    tab.count = 0;
    return launched();
  };
  for (int i = 0; i < count; i++) {
    const int64_t most = (int64_t)1 << 31;
    const int width = dtypes[i] == MXS_DTYPE_F32 ? 4 : 2;
    for (int64_t at = 0; at < sizes[i]; at += most) {
      const int64_t n = sizes[i] - at < most ? sizes[i] - at : most;
      const int chunks = (int)((n + kNormChunk - 1) / kNormChunk);
      if (tab.count == NormTable::N || tab.start[tab.count] > (1 << 30)) {
        const int rc = flush();
        if (rc != MXS_OK) return rc;
      }
      const char* g = static_cast<const char*>(grads[i]) + at * width;
      tab.g[tab.count] = g;
      tab.n[tab.count] = (uint32_t)n;
      tab.flags[tab.count] = (uint8_t)(dtypes[i] | (on16(g) ? kVec : 0));
      tab.start[tab.count + 1] = tab.start[tab.count] + chunks;
      tab.count++;
    }
  }
  const int rc = flush();
  if (rc != MXS_OK) return rc;
  hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(1024), 0, stream, partial, groups, grad_scale,
                     out);
  return launched();
}

int64_t mxs_adamw_workspace_bytes(int count, const int64_t* sizes) {
  if (count < 0 || (count && !sizes)) return MXS_ERR_ARG;
  for (int i = 0; i < count; i++)
    if (sizes[i] < 0) return MXS_ERR_ARG;
  return 64 + (int64_t)sizeof(StepTensor8) * step_entries(count, sizes);
}

int mxs_adamw_step(int count, void* const* params, const void* const* grads, void* const* avgs,
                   void* const* avg_sqs, float* const* avg_scales, float* const* avg_sq_scales,
                   const int64_t* sizes, const int* dtypes, int state_bits, float* step, double lr,
                   const float* lr_dev, double beta1, double beta2, double eps,
                   double weight_decay, const float* norm, double max_norm,
                   const float* grad_scale, const float* found_inf, void* workspace,
                   hipStream_t stream) {
  const bool bits8 = state_bits == 8;
  if (state_bits != 8 && state_bits != 32) return MXS_ERR_DTYPE;
  if (count < 0 || !step || !workspace) return MXS_ERR_ARG;
  if (count && (!params || !grads || !avgs || !avg_sqs || !sizes || !dtypes)) return MXS_ERR_ARG;
  if (count && bits8 && (!avg_scales || !avg_sq_scales)) return MXS_ERR_ARG;
  if ((uintptr_t)workspace % 8) return MXS_ERR_ALIGN;
  for (int i = 0; i < count; i++) {
    if (sizes[i] < 0) return MXS_ERR_ARG;
    if (!dtype_ok(dtypes[i])) return MXS_ERR_DTYPE;
    if (sizes[i] && (!params[i] || !grads[i] || !avgs[i] || !avg_sqs[i])) return MXS_ERR_ARG;
    if (sizes[i] && bits8 && (!avg_scales[i] || !avg_sq_scales[i])) return MXS_ERR_ARG;
  }
  if (step_entries(count, sizes) > (1 << 30)) return MXS_ERR_SIZE;
  StepScalars* scalars = static_cast<StepScalars*>(workspace);
  char* table = static_cast<char*>(workspace) + 64;
  const StepInputs in = {step, lr, lr_dev, beta1, beta2, weight_decay, norm, max_norm, grad_scale,
                         found_inf};
  bool first = true;
  auto base = [&](auto& t, int i, int64_t at) {
    const int64_t wide = dtypes[i] == MXS_DTYPE_F32 ? 4 : 2, state = bits8 ? 1 : 4;
    t.p = static_cast<char*>(params[i]) + at * wide;
    t.g = static_cast<const char*>(grads[i]) + at * wide;
    t.m = static_cast<char*>(avgs[i]) + at * state;
    t.v = static_cast<char*>(avg_sqs[i]) + at * state;
    return on16(t.p) && on16(t.g) && on16(t.m) && on16(t.v);
  };
  auto of_dtype = [&](auto zero, int dtype) {
    using T = decltype(zero);
    if (!bits8)
      return run_step(
          count, sizes, dtypes, dtype, kStepChunk, reinterpret_cast<StepTensor*>(table), scalars,
          first, in, stream, base, [&](const StepTensor* tab, int n, uint32_t chunks) {
            hipLaunchKernelGGL(k_adamw<T>, dim3(chunks), dim3(256), 0, stream, tab, n, scalars,
                               (float)beta1, (float)beta2, (float)(1.0 - beta1),
                               (float)(1.0 - beta2), (float)eps);
          });
    return run_step(
        count, sizes, dtypes, dtype, kStep8Chunk, reinterpret_cast<StepTensor8*>(table), scalars,
        first, in, stream,
        [&](StepTensor8& t, int i, int64_t at) {
          t.ms = avg_scales[i] + at / kStateBlock;
          t.vs = avg_sq_scales[i] + at / kStateBlock;
          return base(t, i, at);
        },
        [&](const StepTensor8* tab, int n, uint32_t chunks) {
          hipLaunchKernelGGL(k_adamw8<T>, dim3(chunks < kStep8Groups ? chunks : kStep8Groups), dim3(256), 0,
                             stream, tab, n, chunks, scalars, beta1, beta2, (float)eps);
        });
  };
  // tensors of one type after the other, over the same table: launches run in order
  int rc = of_dtype(0.0f, MXS_DTYPE_F32);
  if (rc == MXS_OK) rc = of_dtype((_Float16)0, MXS_DTYPE_F16);
  if (rc == MXS_OK) rc = of_dtype((__bf16)0, MXS_DTYPE_BF16);
  if (rc == MXS_OK && first) {  // no values at all: only the step counts
    hipLaunchKernelGGL(k_adamw_setup<StepTensor>, dim3(1), dim3(256), 0, stream,
                       StepPart<StepTensor>{}, 0, reinterpret_cast<StepTensor*>(table), scalars,
                       in);
    rc = launched();
  }
  return rc;
}

int mxs_state_values(const void* codes, const float* scale, int64_t n, int is_signed, float* out,
                     hipStream_t stream) {
  if (n < 0) return MXS_ERR_ARG;
  if (n == 0) return MXS_OK;
  if (!codes || !scale || !out) return MXS_ERR_ARG;
  const int vec = (uintptr_t)codes % 4 == 0 && on16(out);
  for (int64_t at = 0; at < n; at += (int64_t)1 << 34) {  // a launch has fewer than 2^32 lanes
    const int64_t some = n - at < ((int64_t)1 << 34) ? n - at : (int64_t)1 << 34;
    hipLaunchKernelGGL(k_state_values, dim3((unsigned)((some + 4095) / 4096)), dim3(256), 0,
                       stream, static_cast<const uint8_t*>(codes) + at, scale + at / kStateBlock,
                       out + at, some, is_signed ? 0 : 1, vec);
    const int rc = launched();
    if (rc != MXS_OK) return rc;
  }
  return MXS_OK;
}

}  // extern "C"
