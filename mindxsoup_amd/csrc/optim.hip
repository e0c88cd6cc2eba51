// The end of a training step on gfx950: the global 2-norm of many gradient tensors, and the AdamW
// step over many parameter tensors with its two states in fp32 or in 8 bits.
//
// All of it is bound by HBM: every gradient, parameter and state is read once and written once.
// Tensors travel to a launch in its kernel arguments (pointers and sizes, at most 4 KB, so 86
// fp32-state or 63 8-bit-state tensors a launch; 228 gradients of a norm), so a step copies
// nothing to the device and can be captured: a workgroup finds its tensor by a binary search over
// the first chunk of each.
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
constexpr int kStepArgs = 3900;   // bytes of a launch's tensor table

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

struct StepTensor {
  void* p;
  const void* g;
  void *m, *v;
  int64_t n;
};
struct StepTensor8 : StepTensor {
  float *ms, *vs;
};

// Tensors of one launch; flags: dtype (MXS_DTYPE_*) and kVec.
constexpr int kVec = 16;
template <typename T>
struct Table {
  static constexpr int N = (kStepArgs - 8) / (sizeof(T) + 5);
  T t[N];
  int start[N + 1];  // chunks of tensor i: [start[i], start[i + 1])
  uint8_t flags[N];
  int count;
};

// Gradients of one launch of the norm; a longer one than 2^31 values takes several entries.
struct NormTable {
  static constexpr int N = (kStepArgs - 8) / 17;
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

__global__ void k_adamw_scalars(StepScalars* out, float* step, double lr, const float* lr_dev,
                                double beta1, double beta2, double weight_decay,
                                const float* norm, double max_norm, const float* grad_scale,
                                const float* found_inf) {
  const int skip = found_inf && found_inf[0] != 0.0f;
  const float t = step[0] + 1.0f;
  if (lr_dev) lr = (double)lr_dev[0];
  double coef = 1.0;
  if (norm) {
    coef = max_norm / ((double)norm[0] + 1e-6);
    if (coef > 1.0) coef = 1.0;  // a NaN stays one
  }
  if (grad_scale) coef /= (double)grad_scale[0];
  out->coef = coef;
  out->keep = (float)(1.0 - lr * weight_decay);
  out->size = (float)(lr / (1.0 - pow(beta1, (double)t)));
  out->root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
  out->skip = skip;
  if (!skip) step[0] = t;
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
__global__ __launch_bounds__(256) void k_adamw(Table<StepTensor> tab, const StepScalars* scalars,
                                               float b1, float b2, float c1, float c2,
                                               float eps) {
  const StepScalars s = *scalars;
  if (s.skip) return;
  const int c = (int)blockIdx.x, i = tensor_of(tab, c);
  const int64_t at = (int64_t)(c - tab.start[i]) * kStepChunk + threadIdx.x * 8;
  const StepTensor& t = tab.t[i];
  if (at >= t.n) return;
  const bool vec = tab.flags[i] & kVec;
  switch (tab.flags[i] & (kVec - 1)) {
    case MXS_DTYPE_F16: step32<_Float16>(t, at, vec, s, b1, b2, c1, c2, eps); break;
    case MXS_DTYPE_BF16: step32<__bf16>(t, at, vec, s, b1, b2, c1, c2, eps); break;
    default: step32<float>(t, at, vec, s, b1, b2, c1, c2, eps);
  }
}

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

// FULL: all eight values are in the tensor and its pointers are aligned.
template <typename T, bool FULL>
__device__ __forceinline__ void step8(const StepTensor8& t, int64_t i, bool vec,
                                      const StepScalars& s, const Book* books, double b1,
                                      double b2, float eps) {
  // Products and sums rounded one by one: (9 x + y) / 10 of numbers as short as these can lie
  // half way between two fp32 scales, where a fused sum would decide otherwise than the formula.
#pragma clang fp contract(off)
  float p[8], g[8];
  int cm[8], cv[8];
  T* tp = static_cast<T*>(t.p);
  uint8_t *tm = static_cast<uint8_t*>(t.m), *tv = static_cast<uint8_t*>(t.v);
  const int64_t blk = i / kStateBlock, n = FULL ? i + 8 : t.n;
  vec |= FULL;
  load8(static_cast<const T*>(t.g), i, n, vec, g);
  load8_codes(tm, i, n, vec, cm);
  load8_codes(tv, i, n, vec, cv);
  load8(tp, i, n, vec, p);
  const bool any = FULL || blk * kStateBlock < n;
  const double sm = any ? (double)t.ms[blk] : 0.0, sv = any ? (double)t.vs[blk] : 0.0;
  const double d1 = 1.0 - b1, d2 = 1.0 - b2;
  double m[8], v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const double x = (double)g[e] * s.coef;
    const bool in = FULL || i + e < n;
    m[e] = in ? books[0].value[cm[e]] * sm * b1 + x * d1 : 0.0;
    v[e] = in ? books[1].value[cv[e]] * sv * b2 + (x * x) * d2 : 0.0;
    p[e] = p[e] * s.keep - s.size * ratio((float)m[e], (float)v[e], s.root, eps);
  }
  const float topm = encode<true>(books[0], m, cm), topv = encode<false>(books[1], v, cv);
  if (FULL || i < n) {
    store8(tp, i, n, vec, p);
    store8_codes(tm, i, n, vec, cm);
    store8_codes(tv, i, n, vec, cv);
  }
  if (any && (threadIdx.x & 31) == 0) {
    t.ms[blk] = topm;
    t.vs[blk] = topv;
  }
}

template <typename T>
__device__ __forceinline__ void step8_of(const StepTensor8& t, int64_t i, bool vec,
                                         const StepScalars& s, const Book* books, double b1,
                                         double b2, float eps) {
  const int64_t end = i - threadIdx.x % 64 * 8 + 512;  // the wave's
  if (vec && end <= t.n) step8<T, true>(t, i, true, s, books, b1, b2, eps);
  else step8<T, false>(t, i, vec, s, books, b1, b2, eps);
}

__device__ __forceinline__ void books_to_lds(Book* books) {
  const uint32_t* src = reinterpret_cast<const uint32_t*>(kBooks);
  uint32_t* dst = reinterpret_cast<uint32_t*>(books);
  for (int i = threadIdx.x; i < (int)(2 * sizeof(Book) / 4); i += blockDim.x) dst[i] = src[i];
  __syncthreads();
}

// 8-bit states, one pass: 10 bytes a value with 16-bit parameters, 16 with fp32 ones.
__global__ __launch_bounds__(256) void k_adamw8(Table<StepTensor8> tab,
                                                const StepScalars* scalars, double b1, double b2,
                                                float eps) {
  __shared__ Book books[2];
  const StepScalars s = *scalars;
  if (s.skip) return;
  books_to_lds(books);
  for (int c = (int)blockIdx.x; c < tab.start[tab.count]; c += (int)gridDim.x) {
    const int i = tensor_of(tab, c);
    const int64_t at = (int64_t)(c - tab.start[i]) * kStep8Chunk + threadIdx.x * 8;
    const StepTensor8& t = tab.t[i];
    const bool vec = tab.flags[i] & kVec;
    switch (tab.flags[i] & (kVec - 1)) {
      case MXS_DTYPE_F16: step8_of<_Float16>(t, at, vec, s, books, b1, b2, eps); break;
      case MXS_DTYPE_BF16: step8_of<__bf16>(t, at, vec, s, books, b1, b2, eps); break;
      default: step8_of<float>(t, at, vec, s, books, b1, b2, eps);
    }
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

// Puts one tensor after the other into a table and calls launch(table, chunks, chunks before it)
// whenever it is full or holds 2^30 chunks' worth, and at the end.
template <typename T, typename Fill, typename Launch>
static int tables(int count, const int64_t* sizes, int64_t chunk, Fill fill, Launch launch) {
  Table<T> tab;
  tab.count = 0;
  tab.start[0] = 0;
  int64_t before = 0;
  for (int i = 0; i <= count; i++) {
    const int64_t chunks = i < count ? (sizes[i] + chunk - 1) / chunk : 0;
    const bool full = tab.count == Table<T>::N || tab.start[tab.count] + chunks > (1 << 30);
    if (tab.count && (i == count || full)) {
      const int rc = launch(tab, tab.start[tab.count], before);
      if (rc != MXS_OK) return rc;
      before += tab.start[tab.count];
      tab.count = 0;
    }
    if (chunks > (1 << 30)) return MXS_ERR_SIZE;
    if (i == count || chunks == 0) continue;
    fill(tab.t[tab.count], tab.flags[tab.count], i);
    tab.start[tab.count + 1] = tab.start[tab.count] + (int)chunks;
    tab.count++;
  }
  return MXS_OK;
}

static int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MXS_OK : (int)e;
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
  StepScalars* scalars = static_cast<StepScalars*>(workspace);
  hipLaunchKernelGGL(k_adamw_scalars, dim3(1), dim3(1), 0, stream, scalars, step, lr, lr_dev,
                     beta1, beta2, weight_decay, norm, max_norm, grad_scale, found_inf);
  int rc = launched();
  if (rc != MXS_OK) return rc;
  auto flags_of = [&](int i) {
    const bool vec = on16(params[i]) && on16(grads[i]) && on16(avgs[i]) && on16(avg_sqs[i]);
    return (uint8_t)(dtypes[i] | (vec ? kVec : 0));
  };
  if (!bits8)
    return tables<StepTensor>(
        count, sizes, kStepChunk,
        [&](StepTensor& t, uint8_t& flags, int i) {
          t = {params[i], grads[i], avgs[i], avg_sqs[i], sizes[i]};
          flags = flags_of(i);
        },
        [&](const Table<StepTensor>& tab, int chunks, int64_t) {
          hipLaunchKernelGGL(k_adamw, dim3(chunks), dim3(256), 0, stream, tab, scalars,
                             (float)beta1, (float)beta2, (float)(1.0 - beta1),
                             (float)(1.0 - beta2), (float)eps);
          return launched();
        });
  return tables<StepTensor8>(
      count, sizes, kStep8Chunk,
      [&](StepTensor8& t, uint8_t& flags, int i) {
        t.p = params[i], t.g = grads[i], t.m = avgs[i], t.v = avg_sqs[i], t.n = sizes[i];
        t.ms = avg_scales[i], t.vs = avg_sq_scales[i];
        flags = flags_of(i);
      },
      [&](const Table<StepTensor8>& tab, int chunks, int64_t) {
        const int grid = chunks < 2048 ? chunks : 2048;
        hipLaunchKernelGGL(k_adamw8, dim3(grid), dim3(256), 0, stream, tab, scalars, beta1, beta2,
                           (float)eps);
        return launched();
      });
}

int mxs_state_values(const void* codes, const float* scale, int64_t n, int is_signed, float* out,
                     hipStream_t stream) {
  if (n < 0) return MXS_ERR_ARG;
  if (n == 0) return MXS_OK;
  if (!codes || !scale || !out) return MXS_ERR_ARG;
  const int vec = (uintptr_t)codes % 4 == 0 && on16(out);
  for (int64_t at = 0; at < n; at += (int64_t)1 << 40) {  // a grid's 32 bits of workgroups
    const int64_t some = n - at < ((int64_t)1 << 40) ? n - at : (int64_t)1 << 40;
    hipLaunchKernelGGL(k_state_values, dim3((unsigned)((some + 4095) / 4096)), dim3(256), 0,
                       stream, static_cast<const uint8_t*>(codes) + at, scale + at / kStateBlock,
                       out + at, some, is_signed ? 0 : 1, vec);
    const int rc = launched();
    if (rc != MXS_OK) return rc;
  }
  return MXS_OK;
}

}  // extern "C"
