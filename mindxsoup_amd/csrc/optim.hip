// The end of a training step on gfx950: the global 2-norm of many gradient tensors, and the AdamW
// step over many parameter tensors with its two states in fp32 or in 8 bits.
//
// All of it is bound by HBM: every gradient, parameter and state is read once and written once.
// Tensors travel to a launch in its kernel arguments (pointers and sizes, at most 4 KB, so 88
// fp32-state or 64 8-bit-state tensors a launch; 200 gradients of a norm), so a step copies
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
struct Book {
  float value[256];
  double border[256];  // border[c]: a value above it is nearer to code c + 1; [255] is infinite
  // codes to start the search from, by the leading 6 bits of fraction and the exponent of |x|
  uint8_t pos[1474], neg[1474];
};

constexpr int kKeyBase = 104 << 6;          // 2^-23: no border lies between 0 and it
constexpr int kKeys = ((127 - 104) << 6) + 1;  // up to 1
constexpr int kBookSteps = 3;               // borders that a key's interval can hold, and slack

constexpr Book make_book(bool is_signed) {
  Book b{};
  constexpr double decade[7] = {1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 1e-1, 1.0};
  int at = is_signed ? 127 : 0;  // index of zero
  const int zero = at;
  b.value[at++] = 0.0f;
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
  b.value[255] = 1.0f;
  for (int c = 0; c < 255; c++) b.border[c] = ((double)b.value[c] + (double)b.value[c + 1]) / 2;
  b.border[255] = __builtin_huge_val();
  // Interval k of |x|: [lo, hi).  The start is the number of borders surely below x; a hair of
  // slack covers the rounding of x to fp32 before its key is taken.
  double lo = 0.0, scale = 1.0 / (1 << 23);
  int c = 0;
  for (int k = 0; k < kKeys; k++) {
    const double hi = scale * (1.0 + ((k & 63) + 1) / 64.0);
    while (b.border[c] < lo * (1 - 1e-6)) c++;
    b.pos[k] = (uint8_t)c;
    int d = is_signed && c < 254 ? 254 - c : 0;  // symmetric borders but for the one below 1
    while (d > 0 && b.border[d - 1] >= -hi * (1 + 1e-6)) d--;
    b.neg[k] = (uint8_t)d;
    lo = hi;
    if ((k & 63) == 63) scale *= 2;
  }
  return b;
}

// Whether kBookSteps upward steps from every start reach the code of every x of the interval.
constexpr bool book_ok(const Book& b, bool is_signed) {
  double lo = 0.0, scale = 1.0 / (1 << 23);
  for (int k = 0; k < kKeys; k++) {
    const double hi = scale * (1.0 + ((k & 63) + 1) / 64.0);
    if (b.pos[k] && b.border[b.pos[k] - 1] >= lo) return false;
    const int p = b.pos[k] + kBookSteps;
    if (p < 255 && !(b.border[p] >= hi * (1 + 1e-6)) && k + 1 < kKeys) return false;
    if (is_signed) {
      if (b.neg[k] > 127 || (b.neg[k] && b.border[b.neg[k] - 1] >= -hi)) return false;
      const int n = b.neg[k] + kBookSteps;
      if (n < 255 && !(b.border[n] >= -lo * (1 - 1e-6))) return false;
    }
    lo = hi;
    if ((k & 63) == 63) scale *= 2;
  }
  return true;
}

constexpr Book kSignedBook = make_book(true), kUnsignedBook = make_book(false);
static_assert(book_ok(kSignedBook, true) && book_ok(kUnsignedBook, false), "steps of the search");
__device__ __constant__ static const Book kBooks[2] = {kSignedBook, kUnsignedBook};

// The code whose value times `top` is nearest to x (the lower one of two as near): the number of
// borders below x / top.  A border has 25 bits and top 24, so their products are exact; inv,
// about 1 / top, only picks where the search starts.
__device__ __forceinline__ int nearest_code(const Book& b, double x, double top, double inv) {
  const float f = (float)(x * inv);
  int k = (int)((__builtin_bit_cast(uint32_t, f) & 0x7fffffffu) >> 17) - kKeyBase;
  k = min(max(k, 0), kKeys - 1);
  int c = f < 0.0f ? b.neg[k] : b.pos[k];
#pragma unroll
  for (int s = 0; s < kBookSteps; s++) c += b.border[c] * top < x ? 1 : 0;
  return c;
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

struct NormTensor {
  const void* g;
  int64_t n;
};
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

// The tensor of chunk `c` (uniform).
template <typename T>
__device__ __forceinline__ int tensor_of(const Table<T>& tab, int c) {
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

// Sums of squares per chunk, in fp64: the squares of any fp32 and their sums are then neither
// infinite nor lost, whatever their sizes.
__global__ __launch_bounds__(256) void k_norm_chunks(Table<NormTensor> tab, double* partial) {
  __shared__ double s[4];
  const int c = (int)blockIdx.x, i = tensor_of(tab, c);
  const int64_t at = (int64_t)(c - tab.start[i]) * kNormChunk, n = tab.t[i].n;
  const bool vec = tab.flags[i] & kVec;
  double a;
  switch (tab.flags[i] & (kVec - 1)) {
    case MXS_DTYPE_F16: a = squares(static_cast<const _Float16*>(tab.t[i].g), at, n, vec); break;
    case MXS_DTYPE_BF16: a = squares(static_cast<const __bf16*>(tab.t[i].g), at, n, vec); break;
    default: a = squares(static_cast<const float*>(tab.t[i].g), at, n, vec);
  }
  a = sum256(a, s);
  if (threadIdx.x == 0) partial[c] = a;
}

__global__ __launch_bounds__(256) void k_norm_finish(const double* partial, int64_t n,
                                                     const float* grad_scale, float* out) {
  __shared__ double s[4];
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) a += partial[i];
  a = sum256(a, s);
  if (threadIdx.x == 0) out[0] = (float)(sqrt(a) / (grad_scale ? (double)grad_scale[0] : 1.0));
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
    p[e] = p[e] * s.keep - s.size * m[e] / (sqrtf(v[e]) * s.root + eps);
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

// The largest of 32 lanes' values (a block of 256 values lies in half a wave); a NaN wins.
__device__ __forceinline__ float max32(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float y = __shfl_xor(x, o);
    x = (x > y || x != x) ? x : y;
  }
  return x;
}

// New values x[8] of a block as codes and the block's scale.  A block with a value that is not
// finite gets a NaN scale: all of its values are then NaN, as they are lost.
__device__ __forceinline__ float encode(const Book& b, const double (&x)[8], int (&c)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float a = fabsf((float)x[e]);
    top = (top > a || top != top) ? top : a;
  }
  top = max32(top);
  if (top == __builtin_inff()) top = __builtin_nanf("");
  const double inv = top > 0.0f ? 1.0 / (double)top : 0.0;
#pragma unroll
  for (int e = 0; e < 8; e++) c[e] = nearest_code(b, x[e], (double)top, inv);
  return top;
}

template <typename T>
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
  const int64_t blk = i / kStateBlock;
  const bool live = i < t.n;
  load8(static_cast<const T*>(t.g), i, t.n, vec, g);
  load8_codes(tm, i, t.n, vec, cm);
  load8_codes(tv, i, t.n, vec, cv);
  load8(tp, i, t.n, vec, p);
  const bool any = blk * kStateBlock < t.n;
  const double sm = any ? (double)t.ms[blk] : 0.0, sv = any ? (double)t.vs[blk] : 0.0;
  double m[8], v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const double x = (double)g[e] * s.coef;
    const bool in = i + e < t.n;
    m[e] = in ? (double)books[0].value[cm[e]] * sm * b1 + x * (1.0 - b1) : 0.0;
    v[e] = in ? (double)books[1].value[cv[e]] * sv * b2 + (x * x) * (1.0 - b2) : 0.0;
    p[e] = p[e] * s.keep - s.size * (float)m[e] / (sqrtf((float)v[e]) * s.root + eps);
  }
  const float topm = encode(books[0], m, cm), topv = encode(books[1], v, cv);
  if (live) {
    store8(tp, i, t.n, vec, p);
    store8_codes(tm, i, t.n, vec, cm);
    store8_codes(tv, i, t.n, vec, cv);
  }
  if (any && (threadIdx.x & 31) == 0) {
    t.ms[blk] = topm;
    t.vs[blk] = topv;
  }
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
      case MXS_DTYPE_F16: step8<_Float16>(t, at, vec, s, books, b1, b2, eps); break;
      case MXS_DTYPE_BF16: step8<__bf16>(t, at, vec, s, books, b1, b2, eps); break;
      default: step8<float>(t, at, vec, s, books, b1, b2, eps);
    }
  }
}

// The values that codes stand for: book value times scale, rounded once.
__global__ __launch_bounds__(256) void k_state_values(const uint8_t* codes, const float* scale,
                                                      float* out, int64_t n, int book, bool vec) {
  __shared__ float value[256];
  value[threadIdx.x] = kBooks[book].value[threadIdx.x];
  __syncthreads();
  const int64_t stride = (int64_t)gridDim.x * 2048;
  for (int64_t i = (int64_t)blockIdx.x * 2048 + threadIdx.x * 8; i < n; i += stride) {
    int c[8];
    float x[8];
    load8_codes(codes, i, n, vec, c);
    const float s = scale[i / kStateBlock];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = value[c[e]] * s;
    store8(out, i, n, vec, x);
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
  const int rc = tables<NormTensor>(
      count, sizes, kNormChunk,
      [&](NormTensor& t, uint8_t& flags, int i) {
        t = {grads[i], sizes[i]};
        flags = (uint8_t)(dtypes[i] | (on16(grads[i]) ? kVec : 0));
      },
      [&](const Table<NormTensor>& tab, int chunks, int64_t before) {
        hipLaunchKernelGGL(k_norm_chunks, dim3(chunks), dim3(256), 0, stream, tab,
                           partial + before);
        return launched();
      });
  if (rc != MXS_OK) return rc;
  hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(256), 0, stream, partial,
                     norm_chunks(count, sizes), grad_scale, out);
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
  const int64_t chunks = (n + 2047) / 2048;
  hipLaunchKernelGGL(k_state_values, dim3((unsigned)(chunks < 8192 ? chunks : 8192)), dim3(256),
                     0, stream, static_cast<const uint8_t*>(codes), scale, out, n,
                     is_signed ? 0 : 1, on16(codes) && on16(out));
  return launched();
}

}  // extern "C"
