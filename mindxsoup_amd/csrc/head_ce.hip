// The language-model head with its softmax cross entropy on gfx950: for hidden states h [T, D], a
// table W [V, D] and labels y, the losses l_t = log(sum_v exp(z_tv)) - z_ty of z = h W^T, and the
// gradients dh = dz W and dW = dz^T h of dz = softmax(z) - onehot(y).  The logits never exist as
// a matrix: a product's tile leaves its largest value and its sum of exponentials per row, and,
// where gradients are wanted, its exponentials in 16 bits, for at most kPieceBytes of them at a
// time (a piece of the rows); the gradients are products over those.
//
// Rows whose label is to be ignored are taken out first (k_ce_rows gathers the others), so they cost
// nothing and what they hold (infinities, NaN) reaches nothing.
//
// Bound by MFMA: 2 T V D operations per product (one for the losses, a second and third for dh and
// dW), at few rows by reading the table once.  All three products run on one engine
// (stream_tiles): persistent workgroups of eight waves, direct global -> LDS copies of both
// operands that run ahead over tile borders, so that only the first tile of a workgroup waits for
// its operands, and an epilogue from registers while the next tile's copies land.
#include "common.h"
#include "mxs_nf4.h"

namespace mxs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr int kK = 32;             // reduction step: two MFMAs of 16
constexpr int kWaves = 8;          // of a workgroup, but for narrow tiles of the logits
constexpr int kThreads = 64 * kWaves;
constexpr int kRowPad = 256;       // gathered rows are padded with zeros to a multiple of this
constexpr int kVocabTile = 256;    // vocabulary columns of a logits tile
constexpr int64_t kPieceBytes = (int64_t)1 << 30;  // 16-bit exponentials held at a time

// ---- element types ----------------------------------------------------------------------------

template <typename T>
struct Elem;
// Exponentials relative to a power of two are in (0, 1]: times 2^15 they use fp16's whole range
// (normal down to 2^-29); dz in [-1, 1] is kept times 2^14.
template <>
struct Elem<_Float16> {
  static constexpr float kExpBits = 15.0f, kGradBits = 14.0f;
  static __device__ __forceinline__ float16_t mma(u32x4 a, u32x4 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a),
                                                  __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return pack_f16x2(lo, hi);
  }
};
template <>
struct Elem<__bf16> {
  static constexpr float kExpBits = 0.0f, kGradBits = 0.0f;
  static __device__ __forceinline__ float16_t mma(u32x4 a, u32x4 b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x2 v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
};

// ---- what the kernels of a call share -----------------------------------------------------------

struct RowStat {
  float top;    // whole power of two that the row's exponentials but the label's are relative to
  float inv;    // 1 / sum of 2^(z log2 e - top), the label's included
  float miss;   // 1 - p of the label
  float loss;
};

struct CeArgs {
  const void* h;
  int64_t ldh;
  const void* w;
  int64_t ldw;
  const int64_t* labels;
  int64_t ignore;
  int T, V, D;
  const float* row_grad;
  float* loss;   // [T] or [1]
  float* dh;     // [T, D] or null
  float* dw;     // [V, D] or null
  void* dw_final;      // [V, D] in the element type, and the factor from above
  const float* scale;  // (null: 1)
  int mean, per_row;
  // workspace
  int* count;        // rows with a label
  int* share;        // [2] of dh: shares of the vocabulary, steps of one
  float* gmax;       // largest |row_grad| of them
  int* idx;          // [Tp] their rows in h
  int* lab;          // [Tp] their labels; -1 behind the last, -2 outside the vocabulary
  void* hc;          // [Tp, D] gathered
  RowStat* row;      // [Tp]
  float* zy;         // [Tp] the label's logit
  float2* stat;      // [blocks][piece rows] power of two and sum of a block of columns
  uint32_t* shift;   // [blocks][piece rows] binades from a block's to its row's power of two
  u32x4* e;          // [Vp / 32][piece rows / 32][2][64] fragments of exponentials, then dz
  float* part;       // [shares][rows in whole tiles of dh][D]
  // the piece
  int row0, rows;    // first gathered row, rows (a multiple of kRowPad)
  int first;         // the call's first piece
  int last;          // the call's last piece
  int stat_cols;     // columns of a block of `stat`; 0: a block is what a wave of a workgroup saw
  int blocks;        // of `stat`
  int dh_bm, dh_nx;  // rows of a tile of dh, its column tiles
  int dh_most, cus;  // workgroups of dh at most; compute units
};

__device__ __forceinline__ int piece_rows(const CeArgs& a) {
  return min(max(a.count[0] - a.row0, 0), a.rows);
}

// ---- rows with a label ------------------------------------------------------------------------

constexpr int kGather = 8;  // gathered rows of a workgroup

// Gathers the rows whose label is not `ignore`, in order, and pads with zeros.  Every workgroup
// counts all the labels itself (an L2 read of 8 T bytes; one launch, no waiting on another
// workgroup) and copies its own rows.  Ignored rows get their zeros in loss and dh here.
__global__ __launch_bounds__(256) void k_ce_rows(CeArgs a, int vec) {
  __shared__ int s_sum[4], s_idx[kGather];
  const int t = threadIdx.x, r0 = (int)blockIdx.x * kGather, lane = t & 63, wave = t >> 6;
  const int seg = (a.T + 255) / 256 * 64, t0 = min(wave * seg, a.T), t1 = min(t0 + seg, a.T);
  int n = 0;
  for (int i = t0; i < t1; i += 64)
    n += __popcll(__ballot(i + lane < t1 && a.labels[i + lane] != a.ignore));
  if (lane == 0) s_sum[wave] = n;
  if (t < kGather) s_idx[t] = -1;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < wave; w++) at += s_sum[w];
  if (r0 == 0 && t == 0) a.count[0] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  if (at < r0 + kGather && at + n > r0)
    for (int i = t0; i < t1 && at < r0 + kGather; i += 64) {
      const bool has = i + lane < t1 && a.labels[i + lane] != a.ignore;
      const uint64_t all = __ballot(has);
      const int place = at + __popcll(all & ((1ull << lane) - 1));
      if (has && place >= r0 && place < r0 + kGather) s_idx[place - r0] = i + lane;
      at += __popcll(all);
    }
  __syncthreads();
  if (t < kGather) {
    const int i = s_idx[t];
    int y = -1;
    if (i >= 0) {
      const int64_t l = a.labels[i];
      y = l >= 0 && l < a.V ? (int)l : -2;
    }
    a.idx[r0 + t] = i;
    a.lab[r0 + t] = y;
  }
  const int chunks = a.D / 8;  // 16-byte pieces of a row
  for (int r = wave * 2; r < wave * 2 + 2; r++) {
    const int i = s_idx[r];
    u32x4* out = static_cast<u32x4*>(a.hc) + (int64_t)(r0 + r) * chunks;
    const uint16_t* row = static_cast<const uint16_t*>(a.h) + (int64_t)i * a.ldh;
#pragma unroll 4
    for (int k = lane; k < chunks; k += 64) {
      u32x4 v = {0, 0, 0, 0};
      if (i >= 0) {
        const uint16_t* src = row + 8 * k;
        if (vec) {
          v = *reinterpret_cast<const u32x4*>(src);
        } else {
#pragma unroll
          for (int q = 0; q < 4; q++) v[q] = src[2 * q] | ((uint32_t)src[2 * q + 1] << 16);
        }
      }
      out[k] = v;
    }
  }
  for (int r = 0; r < kGather; r++) {
    const int i = r0 + r;
    if (i >= a.T || a.labels[i] != a.ignore) continue;
    if (a.per_row && a.loss && t == 0) a.loss[i] = 0.0f;
    if (a.dh)
      for (int k = t; k < a.D / 4; k += 256)
        reinterpret_cast<float4_t*>(a.dh + (int64_t)i * a.D)[k] = (float4_t){0, 0, 0, 0};
  }
}
static_assert(kGather == 8, "two rows a wave");

// Largest |row_grad| of the rows with a label: dz is kept relative to it, in fp16's range.
__global__ __launch_bounds__(1024) void k_ce_gmax(CeArgs a) {
  __shared__ float s[1024];
  const int t = threadIdx.x;
  float m = 0.0f;
  for (int i = t; i < a.T; i += 1024)
    if (a.labels[i] != a.ignore) {
      const float g = fabsf(a.row_grad[i]);
      m = (m > g || m != m) ? m : g;
    }
  s[t] = m;
  __syncthreads();
  for (int o = 512; o; o >>= 1) {
    if (t < o) {
      const float g = s[t + o];
      m = (m > g || m != m) ? m : g;
      s[t] = m;
    }
    __syncthreads();
  }
  if (t == 0) a.gmax[0] = m;
}

// ---- the engine -------------------------------------------------------------------------------

// One 1 KB direct copy: 16 bytes per lane from base + off to consecutive LDS addresses.  Inline
// asm, so that the compiler's own waits do not count it; completion is awaited by hand.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy1k(uint32_t lds, const void* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return __builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)));
}

__device__ __forceinline__ u32x2 read_tr(const char* p) {
  typedef __attribute__((address_space(3))) short4_t lds_short4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)p));
}

// Copies of one operand's stage by W waves: pieces of 1 KB, piece wave + W i copy i of a wave.
// Where they do not share out evenly, the waves behind the last piece have one copy less.
template <int BYTES, int W = kWaves>
struct Share {
  static constexpr int PIECES = BYTES / 1024, N = (PIECES + W - 1) / W;
  static constexpr bool kEven = PIECES % W == 0;
  __device__ __forceinline__ static bool mine(int i, int wave) {
    return kEven || i + 1 < N || wave + W * i < PIECES;
  }
};

// An operand [ROWS][kK] whose reduction index is contiguous.  64-byte LDS rows of four 16-byte
// segments, segment s of row r at s ^ (r / 4 % 4): 16 rows of a fragment read then fall on all
// banks.  A fragment: row lane % 32, reduction indexes 8 (lane / 32) .. + 7 of its 16.
template <int ROWS, int W = kWaves>
struct RowTile : Share<ROWS * kK * 2, W> {
  static constexpr int BYTES = ROWS * kK * 2;
  using Share<BYTES, W>::N;
  uint32_t off[N];
  const char* base;

  // rows row0 .. of src, those past `last` repeating it
  __device__ __forceinline__ void tile(const void* src, int64_t ld, int row0, int last, int wave,
                                       int lane) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int row = (wave + W * i) * 16 + (lane >> 2);
      const int seg = (lane & 3) ^ ((row >> 2) & 3);
      off[i] = ((uint32_t)min(row, last - row0) * (uint32_t)ld + seg * 8) * 2;
    }
    base = static_cast<const char*>(src) + (int64_t)row0 * ld * 2;
  }
  __device__ __forceinline__ void copy(uint32_t lds, int k, int i, int wave) const {
    copy1k(lds + (wave + W * i) * 1024, base + (int64_t)k * (kK * 2), off[i]);
  }
  __device__ __forceinline__ static u32x4 read(const char* s, int row0, int kk, int lane) {
    const int row = row0 + (lane & 31);
    const int seg = (2 * kk + (lane >> 5)) ^ ((row >> 2) & 3);
    return *reinterpret_cast<const u32x4*>(s + row * 64 + seg * 16);
  }
};

// An operand [kK][COLS] whose reduction index is the row, read through the transposing LDS read.
// LDS rows of COLS / 8 segments, rotated by four for every row of a group of four (two where the
// row length already puts odd rows on the other half of the banks).  A fragment: column
// lane % 32, reduction indexes 4 h .. + 3 and 8 + 4 h .. + 3 of its 16 (h = lane / 32).
template <int COLS>
struct ColTile : Share<COLS * kK * 2> {
  static constexpr int BYTES = COLS * kK * 2, SEGS = COLS / 8;
  using Share<BYTES>::N;
  static constexpr bool kHalf = COLS % 128 != 0;  // rows 32 banks apart
  int row_[N], seg8[N];
  const char* base;
  int64_t ld2;

  __device__ __forceinline__ static int rot(int row) {
    return kHalf ? ((row >> 1) & 1) * 4 : (row & 3) * 4;
  }
  // columns col0 .. of src (whole segments; those past the end repeat the last one)
  __device__ __forceinline__ void tile(const void* src, int64_t ld, int col0, int cols, int wave,
                                       int lane) {
    ld2 = ld * 2;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int q = (wave + kWaves * i) * 64 + lane;
      const int row = q / SEGS, p = q % SEGS;
      const int seg = (p + SEGS - rot(row) % SEGS) % SEGS;
      row_[i] = row;
      seg8[i] = min(seg * 8, cols - 8 - col0) * 2;
    }
    base = static_cast<const char*>(src) + (int64_t)col0 * 2;
  }
  // rows kK k .. of the operand, those past `last` repeating it
  __device__ __forceinline__ void copy(uint32_t lds, int k, int last, int i, int wave) const {
    const int first = min(k * kK, last);
    const uint32_t off = (uint32_t)min(row_[i], last - first) * (uint32_t)ld2 + seg8[i];
    copy1k(lds + (wave + kWaves * i) * 1024, base + first * ld2, off);
  }
  // byte offset of the lane's four values of reduction row 0 of sub-step 0, column block col0
  __device__ __forceinline__ static int read_at(int col0, int lane) {
    const int r = (lane & 15) >> 2, row = 4 * (lane >> 5) + r;
    const int seg = (col0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1) + rot(r)) % SEGS;
    return row * (COLS * 2) + seg * 16 + (lane & 1) * 8;
  }
  __device__ __forceinline__ static u32x4 read(const char* s, int at, int kk) {
    const char* p = s + at + kk * 16 * (COLS * 2);
    const u32x2 a = read_tr(p), b = read_tr(p + 8 * (COLS * 2));
    return (u32x4){a[0], a[1], b[0], b[1]};
  }
};

// The exponentials' fragments: 1 KB blocks [half][32 rows][8 columns] of 32 rows x 16 columns, a
// lane (half h, row r) holding columns 4 h .. + 3 and 8 + 4 h .. + 3.  This is both what a lane of
// the logits product holds after it, and the operand of dh with the reduction over the
// vocabulary: no transposition anywhere.

// Runs a workgroup's `tiles` tiles of `steps` reduction steps.  P: the operands.
//   enter(q)              copies from now on are of tile q
//   copy(lds, q, k, c)    copy c of P::NCP of step k of tile q into the stage at LDS address lds
//   lean                  this wave has P::NCP - 1 copies a step
//   first(s, kk, j), second(s, kk, i): fragments of sub-step kk of the stage at s
//   fix(f, i)             applied to second's fragment before its products
//   load(s), next()       what fix needs of the step in the stage at s: read, then taken over
//   done(q, acc)          tile q's sums; acc[i][j] = first_j x second_i; whether this wave issued
//                         P::STORES stores or more
// P::NS stages of one 32-deep step each, so that P::NS - 1 steps' copies are under way.  Large
// products, which the card's power bounds (1.6 of 2.4 GHz), take the same time with two stages of
// 64; few rows, which wait for their copies, and stores that drain beside later steps want the
// many stages.  A step's second half is multiplied behind the barrier that
// ends it, over the next step's first reads; the stage that this barrier frees takes the copies
// of the step after P::NS, over that half and the next step's first one.
// Waits count what was issued after the copies they wait for (vmcnt retires in order): the copies
// of P::NS - 2 steps, and behind a tile's end, while those copies were issued before it, its
// stores, which so have some steps' time to drain.
template <typename T, int TM, int TN, typename P>
__device__ __forceinline__ void stream_tiles(P& p, char* smem, int tiles, int steps) {
  constexpr int NS = P::NS, NCP = P::NCP, NRD = TM + TN, NMF = TM * TN, HALF = (NCP + 1) / 2;
  static_assert((NS - 2) * NCP + P::STORES <= 63, "vmcnt is 6 bits");
  float16_t acc[TM][TN];
  u32x4 f1[2][TN], f2[2][TM];
  int ct = 0, ck = 0, cstage = 0;  // the copies' tile, step and stage
  const uint32_t lds0 = lds_addr(smem);
  auto copy = [&](int c) { p.copy(lds0 + cstage * P::STAGE, ct, ck, c); };
  auto advance = [&]() {  // to the next step; the last one is copied again rather than none
    cstage = cstage + 1 == NS ? 0 : cstage + 1;
    if (ck + 1 < steps) ck++;
    else if (ct + 1 < tiles) {
      ct++;
      ck = 0;
      p.enter(ct);
    }
  };
  p.enter(0);
#pragma unroll
  for (int s = 0; s < NS; s++) {
#pragma unroll
    for (int c = 0; c < (s + 1 < NS ? NCP : HALF); c++) copy(c);
    if (s + 1 < NS) advance();
  }
  wait_vmem_all();
  lds_barrier();
  auto read = [&](int set, const char* s, int kk, int e) {
    if (e == 0 || e > TN) {
      const int i = e == 0 ? 0 : e - TN;
      f2[set][i] = p.second(s, kk, i);
    } else {
      f1[set][e - 1] = p.first(s, kk, e - 1);
    }
  };
#pragma unroll
  for (int e = 0; e < NRD; e++) read(0, smem, 0, e);
  p.load(smem);
  p.next();
  // multiply set `set`; read sub-step kk of the stage at s into the other one; copies c0 .. c1 - 1
  auto sub = [&](int set, const char* s, int kk, int c0, int c1) {
    int c = c0;
#pragma unroll
    for (int i = 0; i < TM; i++) p.fix(f2[set][i], i);
#pragma unroll
    for (int e = 0; e < NMF; e++) {
      const int i = e / TN, j = e % TN;
      acc[i][j] = Elem<T>::mma(f1[set][j], f2[set][i], acc[i][j]);
#pragma unroll
      for (int q = e * NRD / NMF; q < (e + 1) * NRD / NMF; q++) read(set ^ 1, s, kk, q);
#pragma unroll
      for (; c < c1 && (e + 1) * (c1 - c0) >= (c - c0 + 1) * NMF; c++) copy(c);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int stage = 0, stored = 0;  // steps whose wait may leave the last tile's stores
  for (int q = 0; q < tiles; q++) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
    for (int k = 0; k < steps; k++) {
      sub(0, smem + stage * P::STAGE, 1, HALF, NCP);
      advance();
      if (stored > 0) {
        stored--;
        if (p.lean) wait_vmcnt<(NS - 2) * (NCP - 1) + P::STORES>();
        else wait_vmcnt<(NS - 2) * NCP + P::STORES>();
      } else {
        if (p.lean) wait_vmcnt<(NS - 2) * (NCP - 1)>();
        else wait_vmcnt<(NS - 2) * NCP>();
      }
      lds_barrier();
      stage = stage + 1 == NS ? 0 : stage + 1;
      p.load(smem + stage * P::STAGE);
      sub(1, smem + stage * P::STAGE, 0, 0, HALF);
      p.next();
    }
    stored = p.done(q, acc) ? NS - 2 : 0;
  }
  wait_vmem_all();  // no copy may land after the workgroup's end
}

// Place of workgroup `b` of n in an order in which each XCD (the hardware deals workgroups to the
// eight of them in turn) takes consecutive places.
__device__ __forceinline__ int xcd_place(int b, int n) {
  const int x = b & 7, j = b >> 3, per = n >> 3, rem = n & 7;
  return x * per + min(x, rem) + j;
}

// ---- logits -----------------------------------------------------------------------------------

// BM rows x BN columns a tile, WM x (W / WM) waves.
template <typename T, int BM, int BN_, int W, int WM, int NS_, bool KEEP, bool RANGE>
struct Logits {
  // a wave's statistics run on over its workgroup's tiles, where nothing needs them per tile
  static constexpr bool RUN = RANGE && !KEEP;
  static constexpr int BN = BN_, WN = W / WM, NS = NS_;
  static constexpr int TM = BM / 32 / WM, TN = BN / 32 / WN;
  static constexpr int COLS = 32 * TN;  // columns of a wave: one block of statistics
  using A = RowTile<BM, W>;
  using B = RowTile<BN, W>;
  static constexpr int STAGE = A::BYTES + B::BYTES, NCP = A::N + B::N;
  // Labels of a tile's rows, copied with its first step: a load in the epilogue would wait for
  // every copy before it.  With two steps a tile at least the copies are (NS + 1) / 2 tiles ahead.
  static constexpr int SLOTS = NS > 6 ? 8 : 4, LDS = NS * STAGE + SLOTS * 1024;
  static_assert((NS + 1) / 2 < SLOTS && A::kEven + B::kEven > 0, "label slots, copies per wave");
  static constexpr int STORES = KEEP ? TM * TN * 2 : 0;  // at least: 16 bytes a lane is the widest
  const CeArgs& a;
  const char* smem;
  A ca;
  B cb;
  int wave, lane, mt, wm0, wn0, m_copy;
  int first_col, end;  // of the workgroup's columns, where it has a range of its own
  float run_top[TM], run_sum[TM];
  bool lean;

  __device__ __forceinline__ Logits(const CeArgs& args, const char* lds) : a(args), smem(lds) {
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    lean = !(A::mine(A::N - 1, wave) && B::mine(B::N - 1, wave));
    wm0 = wave / WN * (BM / WM);
    wn0 = wave % WN * COLS;
  }
  // Tiles in an order that keeps an XCD's 32 workgroups on few operands: groups of four vocabulary
  // tiles, all row tiles of a group one after the other.  The hardware deals workgroups to the
  // XCDs in turn, so the 32 of one take consecutive tiles.  Places past the vocabulary are empty.
  __device__ __forceinline__ int place(int q) const {
    return q * (int)gridDim.x + xcd_place((int)blockIdx.x, (int)gridDim.x);
  }
  // RANGE: there is one row tile only, and the table is shared out evenly, in blocks of COLS
  // columns; a workgroup's last tile is then partly empty, and reads no more than its columns.
  __device__ __forceinline__ void coords(int q, int& v0, int& m) const {
    if constexpr (RANGE) {
      v0 = first_col + q * BN;
      m = 0;
    } else {
      const int at = place(q), g = at / (4 * mt), rest = at - g * 4 * mt;
      v0 = (g * 4 + (rest & 3)) * BN;
      m = rest >> 2;
    }
  }
  __device__ __forceinline__ void enter(int q) {
    int v0;
    coords(q, v0, m_copy);
    ca.tile(a.hc, a.D, a.row0 + m_copy * BM, a.row0 + a.rows - 1, wave, lane);
    cb.tile(a.w, a.ldw, min(v0, end - 1), end - 1, wave, lane);
  }
  __device__ __forceinline__ void copy(uint32_t lds, int q, int k, int c) const {
    // one wave's copy more than NCP: the counted waits then wait for more, not for less
    if (c == 0 && k == 0 && wave == 0)
      copy1k(lds_addr(smem) + NS * STAGE + q % SLOTS * 1024, a.lab + a.row0 + m_copy * BM,
             lane * 16);
    if (c < A::N) {
      if (A::mine(c, wave)) ca.copy(lds, k, c, wave);
    } else {
      if (B::mine(c - A::N, wave)) cb.copy(lds + A::BYTES, k, c - A::N, wave);
    }
  }
  __device__ __forceinline__ u32x4 first(const char* s, int kk, int j) const {
    return B::read(s + A::BYTES, wn0 + 32 * j, kk, lane);
  }
  __device__ __forceinline__ u32x4 second(const char* s, int kk, int i) const {
    return A::read(s, wm0 + 32 * i, kk, lane);
  }
  __device__ __forceinline__ void fix(u32x4&, int) const {}
  __device__ __forceinline__ void load(const char*) const {}
  __device__ __forceinline__ void next() const {}

  // acc[i][j][r]: row 32 i + lane % 32, column 32 j + 8 (r / 4) + 4 (lane / 32) + r % 4.
  __device__ __forceinline__ bool done(int q, float16_t (&acc)[TM][TN]) {
    int v0, m;
    coords(q, v0, m);
    if (v0 >= a.V) return false;
    v0 += wn0;
    if (RANGE && v0 >= end) return false;  // another workgroup's
    const int h = lane >> 5;
    if (v0 + COLS > a.V) {  // columns past the vocabulary
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const bool out = v0 + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3) >= a.V;
#pragma unroll
          for (int i = 0; i < TM; i++)
            if (out) acc[i][j][r] = -__builtin_inff();
        }
    }
    constexpr float kLog2e = 1.44269504088896340736f;
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int row = m * BM + wm0 + 32 * i + (lane & 31);  // of the piece
      const int y = reinterpret_cast<const int*>(  // the label's column of this wave
                        smem + NS * STAGE + q % SLOTS * 1024)[wm0 + 32 * i + (lane & 31)] - v0;
      if (__any(y >= 0 && y < COLS)) {  // the label's logit goes to zy alone
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
          for (int r = 0; r < 16; r++)
            if (y == 32 * j + 8 * (r >> 2) + 4 * h + (r & 3)) {
              a.zy[a.row0 + row] = acc[i][j][r];
              acc[i][j][r] = -__builtin_inff();
            }
      }
      float top = acc[i][0][0];
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, __shfl_xor(top, 32));
      // a whole power of two, finite also where every column is -inf
      top = fmaxf(ceilf(top * kLog2e), -3e38f);
      const float bias = Elem<T>::kExpBits - top;
      float sum = 0.0f;
      u32x4* e = nullptr;
      if constexpr (KEEP)
        e = a.e + ((int64_t)(v0 / kK) * (a.rows / 32) + (row >> 5)) * 128 + lane;
#pragma unroll
      for (int j = 0; j < TN; j++) {
        u32x4 f[2];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, bias));
          const float z = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r + 1], kLog2e, bias));
          sum += x;
          sum += z;
          if constexpr (KEEP) f[r >> 3][(r & 7) >> 1] = Elem<T>::pack(x, z);
        }
        if constexpr (KEEP) {
          u32x4* to = e + (int64_t)j * (a.rows / 32) * 128;
          to[0] = f[0];
          to[64] = f[1];
        }
      }
      sum += __shfl_xor(sum, 32);
      if constexpr (RUN) {
        const float to = fmaxf(run_top[i], top);
        run_sum[i] = run_sum[i] * __builtin_amdgcn_exp2f(run_top[i] - to) +
                     sum * __builtin_amdgcn_exp2f(top - to);
        run_top[i] = to;
      } else {
        if (h == 0) a.stat[(int64_t)(v0 / COLS) * a.rows + row] = make_float2(top, sum);
      }
    }
    return KEEP;
  }
  // RUN: the workgroup's waves joined, a block of statistics each
  __device__ __forceinline__ void finish(char* lds) const {
    float2* s = reinterpret_cast<float2*>(lds);
    __syncthreads();  // the stages are done with
#pragma unroll
    for (int i = 0; i < TM; i++)
      if (lane < 32)
        s[(wave % WN) * BM + wm0 + 32 * i + lane] = make_float2(run_top[i], run_sum[i]);
    __syncthreads();
    for (int r = threadIdx.x; r < BM; r += 64 * W) {
      float top = -3e38f, sum = 0.0f;
      for (int w = 0; w < WN; w++) top = fmaxf(top, s[w * BM + r].x);
      for (int w = 0; w < WN; w++)
        sum += s[w * BM + r].y * __builtin_amdgcn_exp2f(s[w * BM + r].x - top);
      a.stat[(int64_t)blockIdx.x * a.rows + r] = make_float2(top, sum);
    }
  }
};

template <typename T, int BM, int BN, int W, int WM, int NS, bool KEEP, bool RANGE>
__global__ __launch_bounds__(64 * W) void k_ce_logits(CeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using P = Logits<T, BM, BN, W, WM, NS, KEEP, RANGE>;
  P p(a, smem);
  p.mt = (piece_rows(a) + BM - 1) / BM;
  const int g = (int)gridDim.x, wg = p.place(0);
  int tiles = 0;
  p.first_col = 0, p.end = a.V;
  if constexpr (RANGE) {
#pragma unroll
    for (int i = 0; i < P::TM; i++) p.run_top[i] = -3e38f, p.run_sum[i] = 0.0f;
    const int blocks = (a.V + P::COLS - 1) / P::COLS, per = (blocks + g - 1) / g * P::COLS;
    p.first_col = wg * per;
    if (p.mt && p.first_col < a.V) {
      p.end = min(p.first_col + per, a.V);
      tiles = (p.end - p.first_col + P::BN - 1) / P::BN;
    }
  } else {
    const int vt = (a.V + P::BN - 1) / P::BN, places = (vt + 3) / 4 * 4 * p.mt;
    tiles = wg < places ? (places - wg + g - 1) / g : 0;
  }
  if (tiles > 0) stream_tiles<T, P::TM, P::TN>(p, smem, tiles, a.D / kK);
  if constexpr (P::RUN) p.finish(smem);
}

// ---- statistics of a row ----------------------------------------------------------------------

// How dh's reduction over the vocabulary is shared out, for the rows that there are: the number of
// shares that takes the fewest rounds of steps over the compute units, their partial sums' traffic
// counted in.  (The host knows only how many rows there could be: with a quarter of 1024 rows
// ignored its shares would leave a quarter of the compute units idle.)
__device__ __forceinline__ void dh_share(const CeArgs& a, int rows) {
  const int steps = (a.V + kK - 1) / kK, tiles = (rows + a.dh_bm - 1) / a.dh_bm * a.dh_nx;
  int best = 0, shares = 1, per = steps;
  for (int z = 1; z * tiles <= a.dh_most && z <= 64 && (z == 1 || 16 * z <= steps); z++) {
    const int n = (steps + z - 1) / z;
    const int cost = (tiles * z + a.cus - 1) / a.cus * (n + 24) + 2 * z;
    if (z == 1 || cost < best) best = cost, shares = (steps + n - 1) / n, per = n;
  }
  a.share[0] = shares;
  a.share[1] = per;
}

// Rows of a workgroup, over 128 strips of blocks (8, 4, 2 rows: 15, 16, 28 us for 768 rows of 151936
// columns, 17, 16, 18 for 261).
constexpr int kJoinRows = 8;

// Joins the blocks' powers of two and sums, all but the label's.  With the label's exponential q
// times smaller than the rest: log-sum-exp = z_y + log(1 + q), and 1 - p_y = q / (1 + q), which the
// gradient takes, stays exact for a label that is all but certain.  The loss is log-sum-exp rounded
// to fp32, less z_y: the cross entropy of fp32 logits, with its 2^-24 |z| of rounding.
// SHIFT: leaves each block's distance to the row's power of two for dh, in both halves of a word
// and at the place of the exponent in a T.
template <typename T, bool SHIFT>
__global__ __launch_bounds__(1024) void k_ce_join(CeArgs a) {
  __shared__ float2 s_part[16][kJoinRows];
  const int n = piece_rows(a), r = threadIdx.x % kJoinRows, strip = threadIdx.x / kJoinRows;
  if ((int)blockIdx.x * kJoinRows >= n) return;
  const int row = (int)blockIdx.x * kJoinRows + r;
  const int blocks = a.blocks;
  float top = -3e38f, sum = 0.0f;
  auto join = [&](float t, float s) {
    const float to = fmaxf(top, t);
    sum = sum * __builtin_amdgcn_exp2f(top - to) + s * __builtin_amdgcn_exp2f(t - to);
    top = to;
  };
  constexpr int kStrips = 1024 / kJoinRows;
#pragma unroll 4
  for (int b = strip; b < blocks; b += kStrips) {
    const float2 x = a.stat[(int64_t)b * a.rows + row];
    join(x.x, x.y);
  }
#pragma unroll
  for (int o = kJoinRows; o < 64; o <<= 1) join(__shfl_xor(top, o), __shfl_xor(sum, o));
  if ((threadIdx.x & 63) < kJoinRows) s_part[threadIdx.x >> 6][r] = make_float2(top, sum);
  __syncthreads();
  top = -3e38f, sum = 0.0f;
  for (int w = 0; w < 16; w++) join(s_part[w][r].x, s_part[w][r].y);
  if (row >= n) return;
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.dh) dh_share(a, n);
  if constexpr (SHIFT) {
    constexpr int kBits = sizeof(T) == 2 && Elem<T>::kExpBits > 0 ? 10 : 7;
    constexpr float kMost = kBits == 10 ? 31.0f : 255.0f;
    for (int b = strip; b < blocks; b += kStrips) {
      const float d = top - a.stat[(int64_t)b * a.rows + row].x;
      a.shift[(int64_t)b * a.rows + row] = (uint32_t)fminf(d, kMost) * (0x10001u << kBits);
    }
  }
  if (strip) return;
  // the sums are of exponentials times 2^kExpBits
  sum *= __builtin_amdgcn_exp2f(-Elem<T>::kExpBits);
  constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
  const int g = a.row0 + row, y = a.lab[g];
  RowStat st = {top, __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
  if (y >= 0 && !(a.zy[g] > 3.4e38f)) {  // (a logit of +inf: NaN, as its exponential is no number)
    const float d = __builtin_fmaf(a.zy[g], kLog2e, -top);  // label's power of two over the rest's
    const float q = sum * __builtin_amdgcn_exp2f(-d);
    const float more = d < -60.0f ? kLn2 * (log2f(sum) - d) : log1pf(q);
    st.loss = a.zy[g] < -3.4e38f ? more : (a.zy[g] + more) - a.zy[g];
    st.miss = q > 1e30f ? 1.0f : q / (1.0f + q);
    st.inv = 1.0f / (sum + __builtin_amdgcn_exp2f(d));
  }
  a.row[g] = st;
  if (a.per_row && a.loss) a.loss[a.idx[g]] = st.loss;
}

// The sum or mean of the losses, in fp64 and a fixed order, by 256 lanes.
__device__ __forceinline__ void total_loss(const CeArgs& a) {
  __shared__ double s[4];
  const int n = a.count[0];
  double x = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) x += (double)a.row[i].loss;
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x) return;
  x = s[0] + s[1] + s[2] + s[3];
  a.loss[0] = (float)(a.mean ? x / (double)n : x);  // 0 / 0 without labels
}

__global__ __launch_bounds__(256) void k_ce_loss(CeArgs a) { total_loss(a); }

// ---- dz ---------------------------------------------------------------------------------------

// Exponentials -> dz times 2^kGradBits (and row_grad over its largest magnitude), in place: 32
// bytes of traffic per eight values.  Rows behind the last become zeros.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_dz(CeArgs a) {
  const int n = piece_rows(a), tbs = a.rows / 32, live = (n + 255) / 256 * 8;
  const int lane = threadIdx.x & 63, b = threadIdx.x >> 6, tb = (int)blockIdx.x;
  if (tb >= live) return;
  const int row = tb * 32 + (lane & 31), h = lane >> 5, g = a.row0 + row;
  float f = 0.0f, top = 0.0f, at_label = 0.0f;
  int y = -1;
  if (row < n) {
    const RowStat st = a.row[g];
    float scale = __builtin_amdgcn_exp2f(Elem<T>::kGradBits);
    if (a.row_grad)
      scale = a.gmax[0] != 0.0f ? scale * (a.row_grad[a.idx[g]] / a.gmax[0]) : 0.0f;
    y = a.lab[g];
    if (y < 0) scale = __builtin_nanf("");
    f = st.inv * scale;
    at_label = -st.miss * scale;
    top = st.top;
  }
  const int pairs = (a.V + kVocabTile - 1) / kVocabTile * (kVocabTile / 64);
  for (int s = (int)blockIdx.y; s < pairs; s += (int)gridDim.y) {
    const int v0 = s * 64 + b * 16;
    u32x4* p = a.e + ((int64_t)(v0 / kK) * tbs + tb) * 128 + (b & 1) * 64 + lane;
    u32x4 x = *p;
    float w = 0.0f;
    if (row < n && v0 < a.V)
      w = f * __builtin_amdgcn_exp2f(
                  a.stat[(int64_t)(v0 / a.stat_cols) * a.rows + row].x - top -
                  Elem<T>::kExpBits);
    typedef T vec8 __attribute__((ext_vector_type(8)));
    const vec8 e = __builtin_bit_cast(vec8, x);
#pragma unroll
    for (int r = 0; r < 8; r += 2) {
      float lo = 0.0f, hi = 0.0f;
      if (row < n && v0 < a.V) {
        const int v = v0 + 8 * (r >> 2) + 4 * h + (r & 3);
        lo = v == y ? at_label : (float)e[r] * w;
        hi = v + 1 == y ? at_label : (float)e[r + 1] * w;
      }
      x[r >> 1] = Elem<T>::pack(lo, hi);
    }
    *p = x;
  }
}

// ---- dh ---------------------------------------------------------------------------------------

// part[z] [rows, D] = dz W over the z-th share of the vocabulary.  SHIFT: of the exponentials as
// the logits product left them, relative to a power of two per row and block of columns, without
// the label's: a fragment is brought to its row's power of two by subtracting binades from the
// exponents, which is exact, and k_ce_dh_sum does the rest (1 / sum, the label's row of the table).
// dz is then never written: at 1024 tokens of a vocabulary of 151936 k_ce_dz takes 92 us.
template <typename T, int BM, int BN, int WM, int NS_, bool SHIFT>
struct HiddenGrad {
  static constexpr int WN = kWaves / WM, NS = NS_, TM = BM / 32 / WM, TN = BN / 32 / WN;
  using B = ColTile<BN>;
  static constexpr int A_BYTES = BM * kK * 2, S_BYTES = SHIFT ? 1024 : 0;
  using A = Share<A_BYTES>;
  static constexpr int STAGE = A_BYTES + B::BYTES + S_BYTES, NCP = A::N + B::N, STORES = 0;
  static constexpr int LDS = NS * STAGE;
  static_assert(A::kEven + B::kEven > 0, "copies per wave");
  const CeArgs& a;
  B cb;
  const char* ebase;
  int wave, lane, m0, n0, k0, wm0, wn0;
  int64_t part_row;  // of the share's partial sums: row 0 of the piece
  bool lean;
  int at[TN];
  uint32_t now[TM], then[TM];

  __device__ __forceinline__ HiddenGrad(const CeArgs& args) : a(args) {
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    lean = !(A::mine(A::N - 1, wave) && B::mine(B::N - 1, wave));
    wm0 = wave / WN * (BM / WM);
    wn0 = wave % WN * (BN / WN);
#pragma unroll
    for (int j = 0; j < TN; j++) at[j] = B::read_at(wn0 + 32 * j, lane);
  }
  __device__ __forceinline__ void enter(int) {
    cb.tile(a.w, a.ldw, n0, a.D, wave, lane);
    ebase = reinterpret_cast<const char*>(a.e) + (int64_t)(m0 / 32) * 2048;
  }
  __device__ __forceinline__ void copy(uint32_t lds, int, int k, int c) const {
    if (c < A::N) {
      const int blk = wave + kWaves * c;
      if (A::mine(c, wave))
        copy1k(lds + blk * 1024,
               ebase + (int64_t)(k0 + k) * (a.rows / 32) * 2048 + blk * 1024, lane * 16);
      // one wave's copy more than NCP: the counted waits then wait for more, not for less
      if (SHIFT && c == 0 && wave == 0)
        copy1k(lds + A_BYTES + B::BYTES,
               a.shift + (int64_t)((k0 + k) * kK / a.stat_cols) * a.rows + m0, lane * 16);
    } else {
      if (B::mine(c - A::N, wave)) cb.copy(lds + A_BYTES, k0 + k, a.V - 1, c - A::N, wave);
    }
  }
  __device__ __forceinline__ u32x4 first(const char* s, int kk, int j) const {
    return B::read(s + A_BYTES, at[j], kk);
  }
  __device__ __forceinline__ u32x4 second(const char* s, int kk, int i) const {
    return *reinterpret_cast<const u32x4*>(s + (wm0 / 32 + i) * 2048 + kk * 1024 + lane * 16);
  }
  __device__ __forceinline__ void load(const char* s) {
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < TM; i++)
        then[i] = *reinterpret_cast<const uint32_t*>(
            s + A_BYTES + B::BYTES + (wm0 + 32 * i + (lane & 31)) * 4);
    }
  }
  __device__ __forceinline__ void next() {
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < TM; i++) now[i] = then[i];
    }
  }
  __device__ __forceinline__ void fix(u32x4& f, int i) const {
    if constexpr (SHIFT) {
      typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
      const ushort2_t n = __builtin_bit_cast(ushort2_t, now[i]);
#pragma unroll
      for (int q = 0; q < 4; q++) {  // below the smallest normal number: zero
        const uint32_t x = f[q];  // (a bit cast of a vector's element would take the first one)
        f[q] = __builtin_bit_cast(
            uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(ushort2_t, x), n));
      }
    }
  }
  __device__ __forceinline__ bool done(int, float16_t (&acc)[TM][TN]) const {
    float* out = a.part + part_row * a.D;
#pragma unroll
    for (int i = 0; i < TM; i++) {
      float* row = out + (int64_t)(m0 + wm0 + 32 * i + (lane & 31)) * a.D;
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const int d = n0 + wn0 + 32 * j + 8 * g + 4 * (lane >> 5);
          if (d < a.D)
            *reinterpret_cast<float4_t*>(row + d) =
                (float4_t){acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                           acc[i][j][4 * g + 3]};
        }
    }
    return false;
  }
};

// Consecutive places are the column tiles of a row tile, then the row tiles of a share: an XCD's
// 32 workgroups read few shares' operands (1024 tokens: one share, all of its tiles).
template <typename T, int BM, int BN, int WM, int NS, bool SHIFT>
__global__ __launch_bounds__(kThreads) void k_ce_dh(CeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using P = HiddenGrad<T, BM, BN, WM, NS, SHIFT>;
  const int ny = (piece_rows(a) + BM - 1) / BM;
  if (ny == 0) return;
  const int shares = a.share[0], per = a.share[1], all = shares * ny * a.dh_nx;
  if ((int)blockIdx.x >= all) return;
  P p(a);
  const int at = xcd_place((int)blockIdx.x, all), x = at % a.dh_nx, yz = at / a.dh_nx;
  p.m0 = yz % ny * BM;
  p.n0 = x * BN;
  p.k0 = yz / ny * per;
  p.part_row = (int64_t)(yz / ny) * ny * BM;
  const int steps = min((a.V + kK - 1) / kK - p.k0, per);
  stream_tiles<T, P::TM, P::TN>(p, smem, 1, steps);
}

// dh rows = the shares' sum, with the scales, to their places in [T, D].
template <typename T, bool SHIFT>
__global__ __launch_bounds__(256) void k_ce_dh_sum(CeArgs a) {
  const int n = piece_rows(a), row = (int)blockIdx.x - 1;
  if (row < 0) {  // one workgroup sums the losses beside the others' work
    if (blockIdx.y == 0 && a.last && a.loss && !a.per_row) total_loss(a);
    return;
  }
  const int d = ((int)blockIdx.y * 256 + (int)threadIdx.x) * 4;
  if (row >= n || d >= a.D) return;
  float4_t x = {0, 0, 0, 0};
  const float* p = a.part + (int64_t)row * a.D + d;
  const int shares = a.share[0];
  const int64_t next = (int64_t)(n + a.dh_bm - 1) / a.dh_bm * a.dh_bm * a.D;
#pragma unroll 4
  for (int z = 0; z < shares; z++) x += *reinterpret_cast<const float4_t*>(p + z * next);
  const int g = a.row0 + row, i = a.idx[g];
  float f = __builtin_amdgcn_exp2f(-Elem<T>::kGradBits);
  if constexpr (SHIFT) {
    const RowStat st = a.row[g];
    const int y = max(a.lab[g], 0);  // (a label outside the vocabulary: st is NaN)
    typedef T vec4 __attribute__((ext_vector_type(4)));
    const vec4 w = *reinterpret_cast<const vec4*>(static_cast<const T*>(a.w) +
                                                  (int64_t)y * a.ldw + d);
    const float inv = st.inv * __builtin_amdgcn_exp2f(-Elem<T>::kExpBits);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = x[e] * inv - st.miss * (float)w[e];
    f = a.row_grad ? a.row_grad[i] : 1.0f;
  } else {
    if (a.row_grad) f *= a.gmax[0];
  }
  if (a.mean) f /= (float)a.count[0];
#pragma unroll
  for (int e = 0; e < 4; e++) x[e] *= f;
  *reinterpret_cast<float4_t*>(a.dh + (int64_t)i * a.D + d) = x;
}

// ---- dW ---------------------------------------------------------------------------------------

// dW [V, D] (+)= dz^T h over the piece's rows: 256 table rows x BN columns a tile, in fp32.  FINAL:
// of a call's only piece, times the factor from above, in T: written once, where the fp32 sums and
// their rounding would move five times those bytes.  Both operands
// have the reduction (the rows of h) across their LDS rows: transposing reads.  A block of dz holds
// 32 rows; in LDS, row t of half b of column block c lies at place t ^ (4 b + 8 (c % 2)), so that
// the 32 lanes of a read meet all banks.
template <typename T, int BN, int NS_, bool FINAL>
struct TableGrad {
  static constexpr int BM = 256, WM = 4, WN = 2, NS = NS_, TM = 2, TN = BN / 64;
  using B = ColTile<BN>;
  static constexpr int A_BYTES = BM * kK * 2;
  using A = Share<A_BYTES>;
  static constexpr int STAGE = A_BYTES + B::BYTES, NCP = A::N + B::N;
  static constexpr int STORES = TM * TN * (FINAL ? 2 : 4), LDS = NS * STAGE;
  static_assert(A::kEven && B::kEven, "copies per wave");
  static constexpr bool lean = false;
  const CeArgs& a;
  B cb;
  const char* ebase;
  int wave, lane, nt, wm0, wn0;
  float factor;  // of the sums: kGradBits, row_grad's largest, the mean, FINAL: from above
  int at[TN], eat[2][2];

  __device__ __forceinline__ TableGrad(const CeArgs& args) : a(args) {
    factor = __builtin_amdgcn_exp2f(-Elem<T>::kGradBits);
    if (a.row_grad) factor *= a.gmax[0];
    if (a.mean) factor /= (float)max(a.count[0], 1);
    if (FINAL && a.scale) factor *= a.scale[0];
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    wm0 = wave / WN * 64;
    wn0 = wave % WN * (BN / WN);
#pragma unroll
    for (int j = 0; j < TN; j++) at[j] = B::read_at(wn0 + 32 * j, lane);
    const int r = (lane & 15) >> 2, s = lane & 3, c = (lane >> 4) & 1, b = s & 1;
#pragma unroll
    for (int odd = 0; odd < 2; odd++)  // sub-step: rows 16 odd .. of a block
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int t = 16 * odd + 8 * x + 4 * (lane >> 5) + r;
        eat[odd][x] = c * 1024 + b * 512 + (t ^ (4 * b + 8 * c)) * 16 + (s >> 1) * 8;
      }
  }
  __device__ __forceinline__ int place(int q) const {
    return q * (int)gridDim.x + xcd_place((int)blockIdx.x, (int)gridDim.x);
  }
  __device__ __forceinline__ void coords(int q, int& v, int& n) const {
    const int at = place(q);
    v = at / nt;
    n = at - v * nt;
  }
  __device__ __forceinline__ void enter(int q) {
    int v, n;
    coords(q, v, n);
    cb.tile(static_cast<const uint16_t*>(a.hc) + (int64_t)a.row0 * a.D, a.D, n * BN, a.D, wave,
            lane);
    ebase = reinterpret_cast<const char*>(a.e) + (int64_t)v * (BM / kK) * (a.rows / 32) * 2048;
  }
  __device__ __forceinline__ void copy(uint32_t lds, int, int k, int c) const {
    if (c < A::N) {  // block of 16 table rows; 32 rows of h
      const int blk = wave + kWaves * c, swap = 4 * (lane >> 5) + 8 * (blk & 1);
      const uint32_t off = ((lane & 32) + ((lane & 31) ^ swap)) * 16;
      copy1k(lds + blk * 1024,
             ebase + ((int64_t)(blk >> 1) * (a.rows / 32) + k) * 2048 + (blk & 1) * 1024, off);
    } else {
      cb.copy(lds + A_BYTES, k, a.rows - 1, c - A::N, wave);
    }
  }
  __device__ __forceinline__ u32x4 first(const char* s, int kk, int j) const {
    return B::read(s + A_BYTES, at[j], kk);
  }
  __device__ __forceinline__ u32x4 second(const char* s, int kk, int i) const {
    const char* p = s + (wm0 / 32 + i) * 2048;
    const u32x2 x = read_tr(p + eat[kk][0]), y = read_tr(p + eat[kk][1]);
    return (u32x4){x[0], x[1], y[0], y[1]};
  }
  __device__ __forceinline__ void fix(u32x4&, int) const {}
  __device__ __forceinline__ void load(const char*) const {}
  __device__ __forceinline__ void next() const {}
  __device__ __forceinline__ bool done(int q, float16_t (&acc)[TM][TN]) const {
    int v, n;
    coords(q, v, n);
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int row = v * BM + wm0 + 32 * i + (lane & 31), h = lane >> 5;
      const bool out = row >= a.V;
      const int64_t at = (int64_t)row * a.D;
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int d0 = n * BN + wn0 + 32 * j;
        if constexpr (FINAL) {
          // the halves of a wave hold columns 8 g .. + 3 and + 4 .. + 7: exchanged, so that a lane
          // stores eight of them
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            uint32_t own[2][2];
#pragma unroll
            for (int q = 0; q < 2; q++)
#pragma unroll
              for (int e = 0; e < 2; e++)
                own[q][e] = Elem<T>::pack(acc[i][j][4 * (g + q) + 2 * e] * factor,
                                          acc[i][j][4 * (g + q) + 2 * e + 1] * factor);
            const uint32_t x = __shfl_xor(h ? own[0][0] : own[1][0], 32);
            const uint32_t y = __shfl_xor(h ? own[0][1] : own[1][1], 32);
            const u32x4 w = h ? (u32x4){x, y, own[1][0], own[1][1]}
                              : (u32x4){own[0][0], own[0][1], x, y};
            const int d = d0 + 8 * (g + h);
            if (!out && d < a.D)
              *reinterpret_cast<u32x4*>(static_cast<T*>(a.dw_final) + at + d) = w;
          }
        } else {
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const int d = d0 + 8 * g + 4 * h;
            if (out || d >= a.D) continue;
            float4_t x;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = acc[i][j][4 * g + e] * factor;
            if (!a.first) x += *reinterpret_cast<const float4_t*>(a.dw + at + d);
            *reinterpret_cast<float4_t*>(a.dw + at + d) = x;
          }
        }
      }
    }
    return (v + 1) * BM <= a.V && (n + 1) * BN <= a.D;  // else some stores fall away
  }
};

template <typename T, int BN, int NS, bool FINAL>
__global__ __launch_bounds__(kThreads) void k_ce_dw(CeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using P = TableGrad<T, BN, NS, FINAL>;
  P p(a);
  p.nt = (a.D + BN - 1) / BN;
  const int places = (a.V + P::BM - 1) / P::BM * p.nt, g = (int)gridDim.x;
  const int wg = p.place(0), tiles = wg < places ? (places - wg + g - 1) / g : 0;
  const int steps = (piece_rows(a) + kK - 1) / kK;
  if (tiles == 0) return;
  if (steps > 0) {
    stream_tiles<T, P::TM, P::TN>(p, smem, tiles, steps);
  } else if (FINAL || a.first) {  // no row has a label
    float16_t acc[P::TM][P::TN] = {};
    for (int q = 0; q < tiles; q++) p.done(q, acc);
  }
}

// ---- gradients to their type --------------------------------------------------------------------

// out = unit * g (one value, or one per row), rounded once.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_scale(const float* unit, const float* g, int per_row,
                                                  int64_t chunks, int row_chunks, T* out) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < chunks;
       c += (int64_t)gridDim.x * 256) {
    const float f = g[per_row ? c / row_chunks : 0];
    const float4_t x = reinterpret_cast<const float4_t*>(unit)[2 * c];
    const float4_t y = reinterpret_cast<const float4_t*>(unit)[2 * c + 1];
    vec8 o;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      o[e] = (T)(x[e] * f);
      o[4 + e] = (T)(y[e] * f);
    }
    reinterpret_cast<vec8*>(out)[c] = o;
  }
}

// ---- host side --------------------------------------------------------------------------------

static int ce_launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MXS_OK : (int)e;
}

// Compute units of the current device (its workgroups fill them one each).
static int ce_cus() {
  static int counts[16];
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16) return 256;
  if (counts[dev] == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0)
      n = 256;
    counts[dev] = n;
  }
  return counts[dev];
}

template <typename K>
static int ce_lds(K fn, int bytes, bool (&set)[16]) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = -1;
  if (dev >= 0 && dev < 16 && set[dev]) return MXS_OK;  // idempotent: a benign race
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return (int)e;
  if (dev >= 0 && dev < 16) set[dev] = true;
  return MXS_OK;
}

// How a call runs: pieces of the rows, tiles.
struct CePlan {
  int Tp, rows, pieces;   // padded rows, rows of a piece
  int bm;                 // rows of a logits tile
  bool narrow;            // of 64 columns instead of 256
  int stat_cols, blocks;
  int dh_bm, dh_bn;
  int64_t part_rows;      // of partial sums of dh
  int64_t vp;             // vocabulary in whole tiles
};

static CePlan ce_plan(int T, int V, int D, bool grads, int cus) {
  CePlan p;
  p.Tp = (T + kRowPad - 1) / kRowPad * kRowPad;
  p.vp = (int64_t)((V + kVocabTile - 1) / kVocabTile) * kVocabTile;
  int64_t most = kRowPad;
  if (grads)
    while (2 * most * p.vp * 2 <= kPieceBytes && most < p.Tp && most < 32768) most *= 2;
  else
    while (most < p.Tp && most < 8192) most *= 2;  // 8 KB of statistics a row at 128 K columns
  p.pieces = (int)((p.Tp + most - 1) / most);
  p.rows = (int)((p.Tp / kRowPad + p.pieces - 1) / p.pieces) * kRowPad;
  // Up to 128 rows one tile holds them; past that tiles of 256, or two of 160 or 192 and three of
  // 192, where 256 would be a quarter empty (301 rows, a call: 202 us; with tiles of 256 230).
  p.bm = T <= 32 && !grads ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : p.pieces > 1 ? 256
         : (T > 256 && T <= 320) || (T > 128 && T <= 160) ? 160
         : (T > 320 && T <= 384) || (T > 512 && T <= 576) || (T > 160 && T <= 192) ? 192 : 256;
  // A small table gives a workgroup 64 columns or fewer.  Tiles that wide take a quarter of the LDS
  // a stage, and with more stages under way a step waits less for its operands.  Losses alone, a
  // call, with tiles of 256 columns and with these: 1 row, 5359 columns of 1536: 23.9, 20.6 us;
  // 11 rows, 5359 of 3264: 39.6, 32.7; 128 rows, 16384 of 4096: 77.0, 48.2.
  p.narrow = T <= 128 && V <= 64 * cus;
  if (p.narrow && p.bm == 32) p.bm = 64;
  const bool run = p.bm <= 128 && !grads;
  p.stat_cols = run ? 0 : p.bm == 256 ? 128 : p.bm == 160 || p.narrow ? 32 : 64;
  p.blocks = run ? cus : (V + p.stat_cols - 1) / p.stat_cols;
  // dh: the tile whose rounds over the compute units take least, each step's fixed part and the
  // shares' partial sums counted in
  p.dh_bm = T <= 64 ? 64 : 256;
  const int steps = (V + kK - 1) / kK, rows = p.pieces > 1 ? p.rows : T;
  const int mt = (rows + p.dh_bm - 1) / p.dh_bm;
  double best = 0;
  for (int bn : {256, 192, 128}) {
    if (bn == 192 && p.dh_bm == 64) continue;  // six column blocks do not share out over the waves
    const int tiles = mt * ((D + bn - 1) / bn);
    for (int z = 1; z <= 64 && (z == 1 || (16 * z <= steps && z * tiles <= 2 * cus)); z++) {
      const int per = (steps + z - 1) / z, rounds = (tiles * z + cus - 1) / cus;
      const double cost = rounds * (per * (0.25 + bn / 256.0) + 24) + 0.5 * z * mt;
      if (best == 0 || cost < best) best = cost, p.dh_bn = bn;
    }
  }
  const int nx = (D + p.dh_bn - 1) / p.dh_bn;
  p.part_rows = (int64_t)(mt > 2 * cus / nx ? mt : 2 * cus / nx + 1) * p.dh_bm;
  return p;
}

struct CeLayout {
  int64_t idx, lab, hc, row, zy, stat, shift, e, part, end;
};

static CeLayout ce_layout(const CePlan& p, int D, bool grads, bool dh) {
  CeLayout l;
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  l.idx = take(4LL * p.Tp);
  l.lab = take(4LL * (p.Tp + 256));  // copied in whole KB
  l.hc = take(2LL * p.Tp * D);
  l.row = take(16LL * p.Tp);
  l.zy = take(4LL * p.Tp);
  // (tiles past the vocabulary's last block leave statistics too)
  const int64_t blocks = p.stat_cols ? p.vp / p.stat_cols : p.blocks;
  l.stat = take(8LL * blocks * p.rows);
  l.shift = grads ? take(4LL * blocks * p.rows) : 0;
  l.e = grads ? take(2LL * p.vp * p.rows) : 0;
  l.part = dh ? take(4LL * p.part_rows * D) : 0;
  l.end = at;
  return l;
}

template <typename T, int BM, int BN, int W, int WM, int NS, bool KEEP, bool RANGE>
static int launch_logits(const CeArgs& a, hipStream_t stream) {
  using P = Logits<T, BM, BN, W, WM, NS, KEEP, RANGE>;
  static bool set[16];
  auto* fn = &k_ce_logits<T, BM, BN, W, WM, NS, KEEP, RANGE>;
  const int rc = ce_lds(fn, P::LDS, set);
  if (rc != MXS_OK) return rc;
  hipLaunchKernelGGL(fn, dim3(a.cus), dim3(64 * W), P::LDS, stream, a);
  return ce_launched();
}

template <typename T, int BM, int BN, int WM, int NS, bool SHIFT>
static int launch_dh(const CeArgs& a, const CePlan& p, hipStream_t stream) {
  using P = HiddenGrad<T, BM, BN, WM, NS, SHIFT>;
  static bool set[16];
  auto* fn = &k_ce_dh<T, BM, BN, WM, NS, SHIFT>;
  const int rc = ce_lds(fn, P::LDS, set);
  if (rc != MXS_OK) return rc;
  hipLaunchKernelGGL(fn, dim3(a.dh_most), dim3(kThreads), P::LDS, stream, a);
  return ce_launched();
}

template <typename T, bool FINAL>
static int launch_dw(const CeArgs& a, hipStream_t stream) {
  constexpr int BN = 256, NS = 4;
  using P = TableGrad<T, BN, NS, FINAL>;
  static bool set[16];
  auto* fn = &k_ce_dw<T, BN, NS, FINAL>;
  const int rc = ce_lds(fn, P::LDS, set);
  if (rc != MXS_OK) return rc;
  hipLaunchKernelGGL(fn, dim3(a.cus), dim3(kThreads), P::LDS, stream, a);
  return ce_launched();
}

#define CE_TRY(call)                      \
  do {                                    \
    const int rc_ = (call);               \
    if (rc_ != MXS_OK) return rc_;        \
  } while (0)

template <typename T, bool KEEP>
static int logits_of(const CeArgs& a, const CePlan& p, hipStream_t stream) {
  if (p.narrow)
    return p.bm == 64 ? launch_logits<T, 64, 64, 4, 2, 12, KEEP, true>(a, stream)
                      : launch_logits<T, 128, 64, 8, 4, 10, KEEP, true>(a, stream);
  switch (p.bm) {
    case 32: return launch_logits<T, 32, 256, 8, 1, 8, KEEP, true>(a, stream);
    case 64: return launch_logits<T, 64, 256, 8, 2, 7, KEEP, true>(a, stream);
    case 128: return launch_logits<T, 128, 256, 8, 2, 6, KEEP, true>(a, stream);
    case 160: return launch_logits<T, 160, 256, 8, 1, 5, KEEP, false>(a, stream);
    case 192: return launch_logits<T, 192, 256, 8, 2, 5, KEEP, false>(a, stream);
    default: return launch_logits<T, 256, 256, 8, 4, 4, KEEP, false>(a, stream);
  }
}

template <typename T, bool SHIFT>
static int dh_of(const CeArgs& a, const CePlan& p, hipStream_t stream) {
  if (p.dh_bm == 64)
    return p.dh_bn == 256 ? launch_dh<T, 64, 256, 2, 6, SHIFT>(a, p, stream)
                          : launch_dh<T, 64, 128, 2, 8, SHIFT>(a, p, stream);
  switch (p.dh_bn) {
    case 256: return launch_dh<T, 256, 256, 4, 4, SHIFT>(a, p, stream);
    case 192: return launch_dh<T, 256, 192, 4, 5, SHIFT>(a, p, stream);
    default: return launch_dh<T, 256, 128, 4, 6, SHIFT>(a, p, stream);
  }
}

template <typename T>
static int run_ce(CeArgs a, const CePlan& p, bool keep_dz, hipStream_t stream) {
  const bool want_dz = a.dw || keep_dz, grads = a.dh || want_dz;
  const int cus = a.cus;
  const int vec = (uintptr_t)a.h % 16 == 0 && a.ldh % 8 == 0;
  hipLaunchKernelGGL(k_ce_rows, dim3(p.Tp / kGather), dim3(256), 0, stream, a, vec);
  CE_TRY(ce_launched());
  if (want_dz && a.row_grad) {
    hipLaunchKernelGGL(k_ce_gmax, dim3(1), dim3(1024), 0, stream, a);
    CE_TRY(ce_launched());
  }
  const bool shift = a.dh && !want_dz;
  for (int i = 0; i < p.pieces; i++) {
    a.row0 = i * p.rows;
    a.rows = p.rows < p.Tp - a.row0 ? p.rows : p.Tp - a.row0;
    a.first = i == 0;
    a.last = i + 1 == p.pieces;
    // tiles that there could be; their shares fill the compute units twice at most
    const int live = a.T - a.row0 < a.rows ? a.T - a.row0 : a.rows;
    const int tiles = (live + p.dh_bm - 1) / p.dh_bm * a.dh_nx;
    a.dh_most = tiles > 2 * cus ? tiles : 2 * cus;
    CE_TRY(grads ? (logits_of<T, true>(a, p, stream)) : (logits_of<T, false>(a, p, stream)));
    if (shift)
      hipLaunchKernelGGL((k_ce_join<T, true>), dim3(a.rows / kJoinRows), dim3(1024), 0, stream, a);
    else
      hipLaunchKernelGGL((k_ce_join<T, false>), dim3(a.rows / kJoinRows), dim3(1024), 0, stream, a);
    CE_TRY(ce_launched());
    if (want_dz) {
      const int tbs = a.rows / 32, ys = 4096 / tbs + 1;
      hipLaunchKernelGGL(k_ce_dz<T>, dim3(tbs, ys), dim3(256), 0, stream, a);
      CE_TRY(ce_launched());
      if (a.dw) CE_TRY((launch_dw<T, false>(a, stream)));
    }
    if (a.dh) {
      CE_TRY(shift ? (dh_of<T, true>(a, p, stream)) : (dh_of<T, false>(a, p, stream)));
      const dim3 grid(a.rows + 1, (a.D / 4 + 255) / 256);
      if (shift)
        hipLaunchKernelGGL((k_ce_dh_sum<T, true>), grid, dim3(256), 0, stream, a);
      else
        hipLaunchKernelGGL((k_ce_dh_sum<T, false>), grid, dim3(256), 0, stream, a);
      CE_TRY(ce_launched());
    }
  }
  if (a.loss && !a.per_row && !a.dh) {
    hipLaunchKernelGGL(k_ce_loss, dim3(1), dim3(256), 0, stream, a);
    CE_TRY(ce_launched());
  }
  return MXS_OK;
}

static int ce_sizes(int T, int V, int D) {
  if (T < 0 || V <= 0 || D <= 0) return MXS_ERR_ARG;
  return D % 64 || D > 65536 || T > (1 << 24) || V > (1 << 28) ? MXS_ERR_SIZE : MXS_OK;
}

}  // namespace mxs

using namespace mxs;

extern "C" {

int64_t mxs_head_ce_workspace_bytes(int T, int V, int D, int want_dh, int want_dw) {
  const int rc = ce_sizes(T, V, D);
  if (rc != MXS_OK) return rc;
  const bool grads = want_dh || want_dw;
  return ce_layout(ce_plan(T > 0 ? T : 1, V, D, grads, ce_cus()), D, grads, want_dh != 0).end;
}

int mxs_head_ce_one_piece(int T, int V, int D) {
  const int rc = ce_sizes(T, V, D);
  if (rc != MXS_OK) return rc;
  return ce_plan(T > 0 ? T : 1, V, D, true, ce_cus()).pieces == 1;
}

// The workspace's places.
static void ce_places(CeArgs& a, const CePlan& p, const CeLayout& l, char* ws, int cus) {
  a.count = reinterpret_cast<int*>(ws);
  a.gmax = reinterpret_cast<float*>(ws + 4);
  a.share = reinterpret_cast<int*>(ws + 8);
  a.idx = reinterpret_cast<int*>(ws + l.idx);
  a.lab = reinterpret_cast<int*>(ws + l.lab);
  a.hc = ws + l.hc;
  a.row = reinterpret_cast<RowStat*>(ws + l.row);
  a.zy = reinterpret_cast<float*>(ws + l.zy);
  a.stat = reinterpret_cast<float2*>(ws + l.stat);
  a.shift = reinterpret_cast<uint32_t*>(ws + l.shift);
  a.e = reinterpret_cast<u32x4*>(ws + l.e);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.stat_cols = p.stat_cols, a.blocks = p.blocks, a.cus = cus;
  a.dh_bm = p.dh_bm, a.dh_nx = (a.D + p.dh_bn - 1) / p.dh_bn;
}

int mxs_head_ce(const void* h, int64_t ldh, const void* w, int64_t ldw, const int64_t* labels,
                int T, int V, int D, int dtype, int64_t ignore_index, int reduction,
                const float* row_grad, float* loss, float* dh, float* dw, int keep_dz,
                void* workspace, hipStream_t stream) {
  const int rc = ce_sizes(T, V, D);
  if (rc != MXS_OK) return rc;
  if (dtype != MXS_DTYPE_F16 && dtype != MXS_DTYPE_BF16) return MXS_ERR_DTYPE;
  if (!w || !workspace || (T && (!h || !labels || (!loss && !dh && !dw && !keep_dz))))
    return MXS_ERR_ARG;
  if (reduction < 0 || reduction > 2 || ldh < D || ldw < D) return MXS_ERR_ARG;
  if (T && (dw || keep_dz) && reduction == 0 && !row_grad) return MXS_ERR_ARG;
  if (dw && keep_dz) return MXS_ERR_ARG;
  if ((uintptr_t)w % 16 || ldw % 8 || (uintptr_t)workspace % 256) return MXS_ERR_ALIGN;
  if ((uintptr_t)dh % 16 || (uintptr_t)dw % 16) return MXS_ERR_ALIGN;
  // offsets within a tile are 32 bits
  if (ldw > (1 << 22) || ldh > ((int64_t)1 << 40)) return MXS_ERR_SIZE;
  const int cus = ce_cus();
  const bool grads = dh || dw || keep_dz;
  const CePlan p = ce_plan(T > 0 ? T : 1, V, D, grads, cus);
  if (keep_dz && p.pieces > 1) return MXS_ERR_SIZE;
  const CeLayout l = ce_layout(p, D, grads, dh != nullptr);
  CeArgs a = {};
  a.h = h, a.ldh = ldh, a.w = w, a.ldw = ldw, a.labels = labels, a.ignore = ignore_index;
  a.T = T, a.V = V, a.D = D, a.row_grad = row_grad, a.loss = loss, a.dh = dh, a.dw = dw;
  a.per_row = reduction == 0;
  a.mean = reduction == 2;
  ce_places(a, p, l, static_cast<char*>(workspace), cus);
  return dtype == MXS_DTYPE_F16 ? run_ce<_Float16>(a, p, keep_dz != 0, stream)
                                : run_ce<__bf16>(a, p, keep_dz != 0, stream);
}

int mxs_head_ce_table_grad(const void* workspace, int T, int V, int D, int dtype, int reduction,
                           const float* row_grad, int want_dh, const float* g, void* dw,
                           hipStream_t stream) {
  const int rc = ce_sizes(T, V, D);
  if (rc != MXS_OK) return rc;
  if (dtype != MXS_DTYPE_F16 && dtype != MXS_DTYPE_BF16) return MXS_ERR_DTYPE;
  if (!workspace || !dw || reduction < 0 || reduction > 2) return MXS_ERR_ARG;
  if ((uintptr_t)dw % 16 || (uintptr_t)workspace % 256) return MXS_ERR_ALIGN;
  const int cus = ce_cus();
  const CePlan p = ce_plan(T > 0 ? T : 1, V, D, true, cus);
  if (p.pieces > 1) return MXS_ERR_SIZE;
  CeArgs a = {};
  a.T = T, a.V = V, a.D = D, a.row_grad = row_grad, a.mean = reduction == 2;
  ce_places(a, p, ce_layout(p, D, true, want_dh != 0),
            static_cast<char*>(const_cast<void*>(workspace)), cus);
  a.rows = p.rows, a.first = 1, a.scale = g, a.dw_final = dw;
  return dtype == MXS_DTYPE_F16 ? launch_dw<_Float16, true>(a, stream)
                                : launch_dw<__bf16, true>(a, stream);
}

int mxs_head_ce_grad(const float* unit, const float* g, int per_row, int64_t rows, int cols,
                     int dtype, void* out, hipStream_t stream) {
  if (rows < 0 || cols <= 0) return MXS_ERR_ARG;
  if (dtype != MXS_DTYPE_F16 && dtype != MXS_DTYPE_BF16) return MXS_ERR_DTYPE;
  if (cols % 8) return MXS_ERR_SIZE;
  if (rows == 0) return MXS_OK;
  if (!unit || !g || !out) return MXS_ERR_ARG;
  if ((uintptr_t)unit % 16 || (uintptr_t)out % 16) return MXS_ERR_ALIGN;
  const int64_t chunks = rows * (cols / 8), wgs = (chunks + 255) / 256;
  const dim3 grid((unsigned)(wgs < 8192 ? wgs : 8192));
  if (dtype == MXS_DTYPE_F16)
    hipLaunchKernelGGL(k_ce_scale<_Float16>, grid, dim3(256), 0, stream, unit, g, per_row, chunks,
                       cols / 8, static_cast<_Float16*>(out));
  else
    hipLaunchKernelGGL(k_ce_scale<__bf16>, grid, dim3(256), 0, stream, unit, g, per_row, chunks,
                       cols / 8, static_cast<__bf16*>(out));
  return ce_launched();
}

}  // extern "C"
