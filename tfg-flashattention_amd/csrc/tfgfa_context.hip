// tfgfa_context.hip - attention of several query rows over a paged key-value cache, MI355X (gfx950), bf16 or fp16, head
// dims that are multiples of 8 up to 128, query heads sharing key-value heads: new tokens of a sequence (tfpages_attend),
// and a decode step of sequences that share a prefix (tfpages_decode_shared).
//
//     o_r = sum_{j < L_r} softmax_j(scale q_r . k_j) v_j,   lse_r = log sum_{j < L_r} e^(scale q_r . k_j)
// The rows r that meet the same keys are one job: a key-value head's query heads, times the new tokens of a sequence, or
// times the sequences behind a prefix.  Bound: HBM for few rows (4 D bytes a key, 4 D flops a key and row), the VALU's
// exponentials beside the matrix units for many.
//
// A block is 32 keys by 32 rows, on v_mfma_f32_32x32x16 (layouts as in tfgfa_fwd.hip):
//   S^T[key][row] = K Q^T: lane (h, i) holds 16 keys of row i, so the softmax of a row is two lanes' own registers;
//   O^T[dim][row] += V^T P^T: those 16 values are the B operand as they stand (the keys' order in the contraction is
//   free), V's operand comes by transposing LDS reads.
// K and V rows go from their pages to LDS by direct loads.  Where a page is a multiple of 16 keys, so many have one page: its
// id and address are scalars, and rows past the end are past its descriptor, which gives zeros.  (8 keys at a time the
// scalar unit, which a CU's waves share, was as busy as the VALU: 8192 causal tokens of 16 heads took 178 us for 157.)
// Other pages: each lane has an address, of a row of zeros where there is no key (pages of 8, 24, 40 and 100 keys alike: 2048
// tokens behind 14336 586 us for 510 to 530, 64 sequences on a prefix of 32000 95 for 72, 16 on each of 4 of 700 29.3 for 27.1,
// 4 tokens behind 1020 13.2 for 11.8).  A page id outside the pool gives a
// row of NaN for K, so that NaN reaches the rows that see the key, and zeros for V.
//
// Few rows (up to 64 a job, 32 a workgroup, the two workgroups of a job side by side): each wave streams blocks of its own
// (wave w of W in a workgroup takes blocks w, w + W, ..) through LDS of its own, with no barrier; they are joined through LDS.
// Many rows: four waves of 32 rows share tiles of 64 keys, and store their rows from registers (through LDS 8 prompts take
// 32.0 us for 29.5).  A job's keys may be divided over workgroups, whose parts a second kernel joins.
//
// Hidden keys have weight 0, but 0 times an infinite or NaN value is NaN: a wave whose sums hold NaN at the end takes its
// keys again with products on the VALU that leave weights of 0 out (so the common path checks nothing).  So does a workgroup
// of many rows, whose offsets are in the log2 domain, where one ends at 2^24 or past it: there rounding it moves all weights
// (8192 causal tokens of 16 heads of 64 with such scores: 3.1 ms for 0.16).
//
// Measured from memory, in graphs, us (a copy moves 5.0 TB/s here, a large bf16 product 1290 TFLOP/s):
//   2048 tokens behind 14336, 32 heads on 8 of 128, fp16, lse     522   988 TFLOP/s: the exponentials and sums of a step hide
//                                                                       behind its products but for a fifth
//   8192 causal tokens of 16 heads of 64                          156   886 TFLOP/s: as many exponentials for half the products
//   8 prompts of up to 800 tokens behind up to 224, 25 heads      29.4  8 steps of 64 keys a workgroup on average, against
//                                                                       about 5 us of its first loads and its end
//   8 tokens behind 30000, twice, 32 heads on 8 of 128            50    4.1 TB/s
//   4 tokens behind 1020, 8 times, 25 heads                       11.8  29 MB; 200 workgroups, start and end 5 us
//   64 sequences on a prefix of 32000, 32 heads on 8 of 128       72    2.9 TB/s: 256 rows a key make the prefix 571 TFLOP/s,
//                                                                       one wave a SIMD, waiting for its tiles half the time
//   16 sequences on each of 4 prefixes of 700, 25 heads           27.3  3.2 TB/s, the join of the parts 5 of it
//   8 sequences on a prefix of 900, 12 heads                      10.1  two launches
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tfgfa.h"
#include "tfgfa_device.h"
#include "tfgfa_layout.h"
#include "tfgfa_pages.h"

namespace tfgfa_context {

using tfgfa::Division;
using tfgfa::i32x4;
using tfgfa::Pages;
using tfgfa::Rows;
using tfgfa::Vecs;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxD = 128;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBlock = 32;                    // keys of a block; rows of a wave's tile
constexpr int kGroup = 16;                    // keys whose rows are loaded together: of one page, where pages are multiples
constexpr int kHalfBytes = kBlock * 128;      // K or V of a block, 64 dims
constexpr int kManyRows = kWaves * kBlock;    // rows of a workgroup for many rows
constexpr int kTile = 2 * kBlock;             // keys of its tile
constexpr int kMaxParts = 32;                 // workgroups of a job
constexpr int kOutOfRange = 0x7FFFFFF0;       // a buffer offset past any num_records: the load gives zeros
// Many rows: an offset is no lower, so that scores of -inf have weight 0 beside it.
constexpr float kLowest = -0x1.fffffep127f;

// kHead: weights are 2^(c (s - m)), s a score without the scale, c the scale times log2 e.  A row's offset m puts the
// largest weight at 2^kHead, and moves when one would pass 2^(kHead + kMargin).  fp16 ends at 2^-24: with the largest at
// 2^13, weights are kept to 2^-37 of it.
template <class T>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef bf16x8 v8;
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static constexpr float kHead = 0.f, kMargin = 8.f;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 x, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(x, v2{(__bf16)1.f, (__bf16)1.f}, acc, false);
  }
};
template <>
struct Elem<_Float16> {
  typedef f16x8 v8;
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static constexpr float kHead = 13.f, kMargin = 2.f;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(v2 x, float acc) {
    return __builtin_amdgcn_fdot2(x, v2{(_Float16)1.f, (_Float16)1.f}, acc, false);
  }
};

// The value of the other half's lane, with the own: a row's two lanes.
template <class F>
__device__ __forceinline__ float over_pair(float x, F f) {
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ int divide(int x, Division d) { return (int)(((uint64_t)(uint32_t)x * d.m) >> d.s); }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ const uint32_t kNanRow[kMaxD / 2] = {
#define TFGFA_8(x) x, x, x, x, x, x, x, x
    TFGFA_8(0x7FFF7FFFu), TFGFA_8(0x7FFF7FFFu), TFGFA_8(0x7FFF7FFFu), TFGFA_8(0x7FFF7FFFu),
    TFGFA_8(0x7FFF7FFFu), TFGFA_8(0x7FFF7FFFu), TFGFA_8(0x7FFF7FFFu), TFGFA_8(0x7FFF7FFFu)};
__device__ const uint32_t kZeroRow[kMaxD / 2] = {};

typedef const __attribute__((address_space(4))) int* uniform_ints;

// A sequence's keys in one key-value head.
struct Source {
  const char* k;  // the pools, at the head
  const char* v;
  Pages ks, vs;
  const int* table;
  Division by_page;
  int page, P;
  int keys;       // keys that there are
};

// 1 KiB from 64 addresses to LDS, as tfgfa::lds_transfer does from a buffer.
__device__ __forceinline__ void lds_gather(uint64_t from, uint32_t lds_base) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(lds_base), "v"(from)
      : "memory");
}

__device__ __forceinline__ int swz_v(int row) { return (row & 3) << 1; }

// Two transfers of one buffer, to LDS bytes `first` and `second` (tfgfa::lds_transfer, with one exchange of M0).
__device__ __forceinline__ void lds_pair(i32x4 desc, uint32_t first, int off0, uint32_t second, int off1) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %3, %5, 0 offen lds\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %4, %5, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(first), "s"(second), "v"(off0), "v"(off1), "s"(desc)
      : "memory");
}

// Loads of kGroups groups of 16 keys, from group g0 of a block on.  A block in LDS: K's (or V's) halves of 64 dims, each 32
// rows of 128 bytes; chunk c of row r at place c ^ swz (tfgfa_fwd.hip says why).  Lane l of a transfer fills chunk l % 8
// of row l / 8 of its 8 rows.
template <int kDH, bool kAligned, int kGroups>
struct Loader {
  int koff[kGroups][2][kDH], voff[2][kDH];  // aligned: byte offsets from the group's first row; otherwise in a row, or out of range
  int g0, lane;

  // Where a block's rows are: of each group the page and its row in it, or (not aligned) of key l % 32 in lane l the page.
  struct Place {
    int page[kAligned ? kGroups : 1], row[kAligned ? kGroups : 1];
  };

  __device__ __forceinline__ void init(const Source& s, int D, int g0_, int lane_) {
    g0 = g0_, lane = lane_;
    const int r = lane >> 3, chunks = D >> 3;
#pragma unroll
    for (int dh = 0; dh < kDH; ++dh)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int c = 8 * dh + ((lane & 7) ^ tfgfa::swz_k((g0 + g) * kGroup + 8 * i + r));
          koff[g][i][dh] = c < chunks ? (kAligned ? (8 * i + r) * (int)s.ks.n : 0) + 16 * c : kOutOfRange;
        }
        const int c = 8 * dh + ((lane & 7) ^ swz_v(r));
        voff[i][dh] = c < chunks ? (kAligned ? (8 * i + r) * (int)s.vs.n : 0) + 16 * c : kOutOfRange;
      }
  }
  // The place of the block at key `at`.
  __device__ __forceinline__ Place look_up(const Source& s, int at) const {
    Place x;
    if constexpr (kAligned) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int key = at + (g0 + g) * kGroup, column = divide(key, s.by_page);
        x.page[g] = uniform(key < s.keys ? ((uniform_ints)s.table)[column] : 0);
        x.row[g] = key - column * s.page;
      }
    } else {
      const int key = at + (lane & 31);
      x.page[0] = key < s.keys ? s.table[divide(key, s.by_page)] : 0;
    }
    return x;
  }
  // K (kValue: V) of the block at key `at` to LDS byte `to`.
  template <bool kValue>
  __device__ __forceinline__ void issue(const Source& s, int at, const Place& x, uint32_t to) const {
    const Pages& st = kValue ? s.vs : s.ks;
    const char* const base = kValue ? s.v : s.k;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t there = to + (g0 + g) * 2048;
      if constexpr (kAligned) {
        const int rows = uniform(min(kGroup, max(0, s.keys - at - (g0 + g) * kGroup)));
        const bool in = (uint32_t)x.page[g] < (uint32_t)s.P;
        const uint64_t page = (uint32_t)(in ? x.page[g] : 0), row = (uint32_t)x.row[g];
        const i32x4 desc = tfgfa::head_desc(base + page * (uint64_t)st.p + row * (uint64_t)st.n, uniform(in ? rows : 0), (int)st.n);
        if (kValue || in || rows == 0) {
#pragma unroll
          for (int dh = 0; dh < kDH; ++dh)
            lds_pair(desc, there + dh * kHalfBytes, kValue ? voff[0][dh] : koff[g][0][dh], there + dh * kHalfBytes + 1024,
                     kValue ? voff[1][dh] : koff[g][1][dh]);
        } else {
          const i32x4 nan = tfgfa::head_desc(kNanRow, 1, sizeof(kNanRow));
#pragma unroll
          for (int dh = 0; dh < kDH; ++dh)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = 8 * i + (lane >> 3);
              tfgfa::lds_transfer(nan, there + dh * kHalfBytes + 1024 * i,
                                  koff[g][i][dh] == kOutOfRange || r >= rows ? kOutOfRange : koff[g][i][dh] - r * (int)st.n);
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = (g0 + g) * kGroup + 8 * i + (lane >> 3), key = at + r;
          const int page = __shfl(x.page[0], r);
          const bool seen = key < s.keys, in = seen && (uint32_t)page < (uint32_t)s.P;
          const uint64_t pid = (uint32_t)(in ? page : 0), off = (uint32_t)(in ? key - divide(key, s.by_page) * s.page : 0);
          const uint64_t zero = (uint64_t)(uintptr_t)kZeroRow;
          const uint64_t row = in ? (uint64_t)(uintptr_t)base + pid * (uint64_t)st.p + off * (uint64_t)st.n
                                  : !kValue && seen ? (uint64_t)(uintptr_t)kNanRow : zero;
#pragma unroll
          for (int dh = 0; dh < kDH; ++dh) {
            const int at_lane = kValue ? voff[i][dh] : koff[g][i][dh];
            lds_gather(at_lane == kOutOfRange ? zero : row + at_lane, there + dh * kHalfBytes + 1024 * i);
          }
        }
      }
    }
  }
};

// A wave's 32 rows, row i in lanes i and i + 32.
// kParts: of the element type that a weight is split into for the product with V, each what rounding left of the ones
// before (2: all but 2^-16 of a weight in bf16, 2^-22 in fp16).  With 1 the output is divided by the sum of the rounded
// weights, so that the rounding of a weight that stands alone cancels; the log-sum-exp takes the unrounded ones.
template <class T, int kDH, int kParts>
struct State {
  typedef typename Elem<T>::v8 v8;
  typedef typename Elem<T>::v2 v2;
  static constexpr int kC = 4 * kDH;   // pieces of 16 dims
  static constexpr int kOT = 2 * kDH;  // output tiles of 32
  v8 q[kC];
  f32x16 o[kOT];
  float m, thr;             // offset, and how far a score may pass it (-inf: the row has no weight yet)
  float l, lp;              // this lane's sums of weights, and (kParts 1) of the rounded ones
  int seen;                 // keys that the row sees
  int koff[4], voff[2][2];  // LDS offsets of the operands, in a block's first 64 dims

  __device__ __forceinline__ void init(int lane) {
    const int i = lane & 31, h = lane >> 5, g = lane >> 4, j = lane & 15;
#pragma unroll
    for (int c = 0; c < 4; ++c) koff[c] = i * 128 + (((2 * c + h) ^ tfgfa::swz_k(i)) << 4);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int row = 8 * s + 4 * (g >> 1) + (j >> 2), d = 32 * t + 16 * (g & 1) + 4 * (j & 3);
        voff[t][s] = row * 128 + (((d >> 3) ^ swz_v(row)) << 4) + (d & 7) * 2;
      }
    clear();
  }
  __device__ __forceinline__ void clear() {
    m = l = lp = 0.f, thr = -INFINITY;
#pragma unroll
    for (int j = 0; j < kOT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[j][r] = 0.f;
  }

  // S^T of the block in LDS.
  __device__ __forceinline__ void scores(f32x16& s, const unsigned char* block) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const v8 a = key_operand(block, c);
      s = Elem<T>::mfma(a, q[c], s);
    }
  }

  static __device__ __forceinline__ float largest(const f32x16& s) {
    float x = fmaxf(s[0], fmaxf(s[1], s[2]));
#pragma unroll
    for (int r = 3; r < 15; r += 2) x = fmaxf(fmaxf(x, s[r]), s[r + 1]);
    return fmaxf(x, s[15]);
  }

  // Few rows, and the exact pass: weights 2^(c (s - m)) in place.  (The difference first, which is exact for near
  // scores of any size.)  c: scale_log2.
  __device__ __forceinline__ void weigh(f32x16& s, float c, float inv_c) {
    const float mx = largest(s);
    if (__builtin_amdgcn_ballot_w64(mx - m >= thr)) {
      const float top = over_pair(mx, [](float x, float y) { return fmaxf(x, y); });
      const bool fresh = thr == -INFINITY, none = top == -INFINITY;  // no weight so far; none here
      const float to = none ? m : fmaxf(fresh ? -INFINITY : m, top - fminf(Elem<T>::kHead * inv_c, 1e30f));
      const float f = fresh ? 0.f : __builtin_amdgcn_exp2f((m - to) * c);
      m = to;
      if (!none) thr = fminf((Elem<T>::kHead + Elem<T>::kMargin) * inv_c, 1e30f);
      l *= f, lp *= f;
#pragma unroll
      for (int j = 0; j < kOT; ++j) o[j] *= f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f((s[r] - m) * c);
  }

  // Scores of keys that a row does not see; at: the block's first key.
  __device__ __forceinline__ void mask(f32x16& s, int at, int lane) const {
    const int left = seen - at - 4 * (lane >> 5);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 < left ? s[r] : -INFINITY;
  }

  __device__ __forceinline__ v8 values(const unsigned char* v, int j, int c) const {
    const unsigned char* const at = v + (j >> 1) * kHalfBytes + c * 16 * 128;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(at + voff[j & 1][0]));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(at + voff[j & 1][1]));
    return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // Weights as operands.
  static __device__ __forceinline__ void parts_of(const float* p, v8 (&part)[kParts][2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = p[8 * c + e];
#pragma unroll
        for (int n = 0; n < kParts; ++n) {
          T y;
          if (std::is_same_v<T, __bf16> && n + 1 < kParts)  // cut off: two operations less than rounding, and no part below 0
            y = __builtin_bit_cast(T, (unsigned short)(__float_as_uint(x) >> 16));
          else
            y = (T)x;
          part[n][c][e] = y;
          if (n + 1 < kParts) x -= (float)y;
        }
      }
  }
  static __device__ __forceinline__ float sum16(const float* p) {
    float a = p[0], b = p[1];
#pragma unroll
    for (int r = 2; r < 16; r += 2) a += p[r], b += p[r + 1];
    return a + b;
  }
  // x and the sum of the weights as rounded (of two parts: the first).
  static __device__ __forceinline__ float add_rounded(const v8 (&part)[kParts][2], float x) {
    float y = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      x = Elem<T>::add2(v2{part[0][0][e], part[0][0][e + 1]}, x);
      y = Elem<T>::add2(v2{part[0][1][e], part[0][1][e + 1]}, y);
    }
    return x + y;
  }
  __device__ __forceinline__ void split(const f32x16& w, v8 (&part)[kParts][2]) {
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = w[r];
    l += sum16(p);
    parts_of(p, part);
  }

  // O^T += V^T P^T.
  __device__ __forceinline__ void output(const unsigned char* v, const v8 (&part)[kParts][2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < kOT; ++j) {
        const v8 a = values(v, j, c);
#pragma unroll
        for (int n = 0; n < kParts; ++n) o[j] = Elem<T>::mfma(a, part[n][c], o[j]);
      }
  }

  // The same with float32 products that leave weights of 0 out.
  __device__ __forceinline__ void output_exact(const unsigned char* v, const f32x16& p, int lane) {
    const int h = lane >> 5;
#pragma unroll 1
    for (int r = 0; r < 16; ++r) {
      float x = p[0];
#pragma unroll
      for (int u = 1; u < 16; ++u) x = r == u ? p[u] : x;
      const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      const float both[2] = {__uint_as_float(y[0]), __uint_as_float(y[1])};
      l += x, lp += x;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int key = 8 * (r / 4) + 4 * hh + r % 4;
#pragma unroll
        for (int j = 0; j < kOT; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int d = (32 * j + 8 * g) & 63;
            typedef T v4 __attribute__((ext_vector_type(4)));
            const v4 x = *reinterpret_cast<const v4*>(v + (j >> 1) * kHalfBytes + key * 128 + (((d >> 3) ^ swz_v(key)) << 4) + 8 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = both[hh];
              o[j][4 * g + e] = y == 0.f ? o[j][4 * g + e] : fmaf(y, (float)x[e], o[j][4 * g + e]);
            }
          }
      }
    }
  }

  // One block; at: its first key; least: keys that every row of the wave sees.
  template <bool kExact>
  __device__ __forceinline__ void step(const unsigned char* k, const unsigned char* v, int at, int least, float c, float inv_c,
                                       int lane) {
    f32x16 s;
    scores(s, k);
    if (at + kBlock > least) mask(s, at, lane);
    weigh(s, c, inv_c);
    if constexpr (kExact) {
      output_exact(v, s, lane);
    } else {
      v8 part[kParts][2];
      split(s, part);
      output(v, part);
    }
  }

  // Many rows (kParts 1): blocks in a pipeline.  s: the scores of block u; part: the weights of block u - 1; v, k: V of block
  // u - 1 and K of block u + 1 in LDS.  The products of V run beside the exponentials, those of K beside the weights' sums
  // and rounding, one matrix instruction and a share of them at a time (a wave's VALU work overlaps its own matrix
  // instructions).  Offsets are in the log2 domain (m = thr): 2^(c s - m) is one v_fma and one v_exp.
  // The sum of the rounded weights tells when an offset has to move: a weight past the type's range, or a sum past kBound,
  // is infinite, NaN or above it.
  static constexpr float kBound = std::is_same_v<T, __bf16> ? 0x1p64f : 0x1.fffffep127f;
  template <bool kPV, bool kLse>
  __device__ __forceinline__ void fused(const unsigned char* v, const unsigned char* k, f32x16& s, v8 (&part)[kParts][2],
                                        float c, float head) {
    constexpr int kPairs = 2 * kOT;
    v8 vo[2], ko[2];
    if constexpr (kPV) vo[0] = values(v, 0, 0), vo[1] = values(v, 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    float p[16];
    const float neg = -m;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int cc = i / kOT, j = i % kOT;
      if constexpr (kPV) o[j] = Elem<T>::mfma(vo[i & 1], part[0][cc], o[j]);
      if (i + 2 < kPairs) {
        if constexpr (kPV) vo[i & 1] = values(v, (i + 2) % kOT, (i + 2) / kOT);
      } else {
        ko[i + 2 - kPairs] = key_operand(k, i + 2 - kPairs);
      }
#pragma unroll
      for (int r = 16 * i / kPairs; r < 16 * (i + 1) / kPairs; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, neg));
        asm volatile("" : "+v"(p[r]));  // (here, though the rare branch takes them again)
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x16 next;
#pragma unroll
    for (int r = 0; r < 16; ++r) next[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      next = Elem<T>::mfma(ko[i & 1], q[i], next);
      if (i + 2 < kC) ko[i & 1] = key_operand(k, i + 2);
      if (i == 0) {
        parts_of(p, part);
        asm volatile("" : "+v"(part[0][0]), "+v"(part[0][1]));
      } else if (i == 1) {
        float sum = add_rounded(part, lp);
        // (As integers: past the bound, infinite or NaN.)
        if (__builtin_amdgcn_ballot_w64(__float_as_uint(sum) > __float_as_uint(kBound))) {
          const float top = over_pair(largest(s), [](float x, float y) { return fmaxf(x, y); });
          const float to = fmaxf(fmaxf(m, kLowest), top * c - head);
          const float f = __builtin_amdgcn_exp2f(m - to);
          m = to, lp *= f, l *= f;
#pragma unroll
          for (int j = 0; j < kOT; ++j) o[j] *= f;
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -to));
          parts_of(p, part);
          sum = add_rounded(part, lp);
        }
        lp = sum;
        asm volatile("" : "+v"(lp));
      }
      if (i == 2 && kLse) {
        l += sum16(p);
        asm volatile("" : "+v"(l));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    s = next;
  }
  __device__ __forceinline__ v8 key_operand(const unsigned char* k, int c) const {
    return *reinterpret_cast<const v8*>(k + (c >> 2) * kHalfBytes + koff[c & 3]);
  }

  // Whether some sum of the wave is NaN.
  __device__ __forceinline__ bool any_nan() const {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < kOT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) x = fmaf(o[j][r], 0.f, x);
    return __builtin_amdgcn_ballot_w64(x != x) != 0;
  }

  // Many rows: the offset from the log2 domain to scores without the scale.  What rounding it there leaves, m c - to, goes
  // into the sums, so that it is exact.
  __device__ __forceinline__ void rescale(float c) {
    if (!(fabsf(m) < INFINITY)) return;
    if (m <= kLowest) {  // scores of -inf alone
      m = -INFINITY;
      return;
    }
    const float to = m / c, f = __builtin_amdgcn_exp2f(-fmaf(to, c, -m));
    m = to, l *= f, lp *= f;
#pragma unroll
    for (int j = 0; j < kOT; ++j) o[j] *= f;
  }

  // Few rows (kParts 2), into LDS: rows of 64 kDH floats, 16-byte piece c of row r at place c ^ r % pieces; statistics beside.
  __device__ __forceinline__ void publish(unsigned char* rows, float* sm, float* sl, int lane) const {
    constexpr int kPieces = 16 * kDH;
    const int r = lane & 31, h = lane >> 5;
    const float lt = over_pair(l, [](float x, float y) { return x + y; });
#pragma unroll
    for (int j = 0; j < kOT; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 8 * j + 2 * g + h;
        *reinterpret_cast<f32x4*>(rows + (r * kPieces + (c ^ (r % kPieces))) * 16) =
            f32x4{o[j][4 * g], o[j][4 * g + 1], o[j][4 * g + 2], o[j][4 * g + 3]};
      }
    if (h == 0) sm[r] = thr == -INFINITY ? -INFINITY : m, sl[r] = lt;
  }
};

// A piece of work: rows [row0, row0 + 32 or 128) of a job, blocks [first, last) of its keys.
struct Job {
  const void* q;                  // the job's first row; row r is r / G steps and r % G heads on
  long long q_step, q_head;
  Division by_group;
  int G, row0, rows;              // rows: of the job
  int seen, causal;               // row r sees the keys below seen (+ r / G + 1, causal)
  int first, last;
  float scale, scale_log2;
};

// Where its rows go: the outputs, or (part) its part of them: D floats a row of sums, and of each row the offset and the
// sums of weights, part_rows rows of each (those that there are: 512 sequences of 32 heads of 128 behind a prefix keep 10.5 MB
// of their own, a tile's 32 rows each would be 275).
struct Sink {
  void* o;
  long long o_step, o_head;       // elements
  float* lse;
  long long l_step, l_head;
  float* part;
  int part_rows;
  int fill_to, fill;              // rows from Job::rows up to here get zeros (fill 1) or NaN (fill 2)
};

// Floats of a part: whole lines of 128 bytes.
__host__ __device__ constexpr long long part_floats(int rows, int D) { return ((long long)rows * (D + 3) + 31) / 32 * 32; }

constexpr int few_lds(int kDH, int waves) {  // a block of each wave, or its rows
  const int blocks = waves * 2 * kDH * kHalfBytes, rows = waves * kBlock * 64 * kDH * 4;
  return blocks > rows ? blocks : rows;
}
constexpr int many_lds(int kDH) { return 4 * kDH * 2 * kHalfBytes; }  // four tiles of 64 keys

// Of each wave's rows.
template <int kW>
struct Stats {
  float m[kW * kBlock], l[kW * kBlock];
};

template <class T, int kDH, int kParts>
__device__ __forceinline__ void load_rows(State<T, kDH, kParts>& w, const Job& job, int first, int D, int lane) {
  typedef typename Elem<T>::v8 v8;
  const int r = first + (lane & 31), h = lane >> 5, step = divide(r, job.by_group);
  const T* const at = static_cast<const T*>(job.q) + step * job.q_step + (r - step * job.G) * job.q_head;
  w.seen = r < job.rows ? job.seen + (job.causal ? step + 1 : 0) : 0;
#pragma unroll
  for (int c = 0; c < 4 * kDH; ++c) {
    const int d = 16 * c + 8 * h;
    w.q[c] = __builtin_bit_cast(v8, u32x4{0, 0, 0, 0});
    if (r < job.rows && d < D) w.q[c] = *reinterpret_cast<const v8*>(at + d);
  }
  // Here, before the loop: the waits that the compiler places for these loads would empty the pipeline of direct ones.
#pragma unroll
  for (int c = 0; c < 4 * kDH; ++c) asm volatile("" ::"v"(w.q[c]));
}

// Few rows: row `row` of the workgroup's, 8 dims from 8 c8 on, joined over the waves' states, to its place.
template <class T, int kDH, int kW>
__device__ __forceinline__ void put(const unsigned char* rows, const Stats<kW>& st, int row, int c8, const Job& job,
                                    const Sink& to, int D) {
  constexpr int kPieces = 16 * kDH;
  const int r = job.row0 + row;
  const bool real = r < job.rows;
  if (!real && !(to.part == nullptr && to.fill != 0 && r < to.fill_to)) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kW; ++w) M = fmaxf(M, st.m[w * kBlock + row]);
  float l = 0.f;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    const int at = w * kBlock + row;
    const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m[at] - M) * job.scale_log2);
    l = fmaf(f, st.l[at], l);
    const f32x4 x = *reinterpret_cast<const f32x4*>(rows + (at * kPieces + ((2 * c8) ^ (at % kPieces))) * 16);
    const f32x4 y = *reinterpret_cast<const f32x4*>(rows + (at * kPieces + ((2 * c8 + 1) ^ (at % kPieces))) * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // (a wave without weight has no sums; its offset may be NaN's)
      a[e] = f == 0.f ? a[e] : fmaf(f, x[e], a[e]);
      b[e] = f == 0.f ? b[e] : fmaf(f, y[e], b[e]);
    }
  }
  if (to.part) {
    float* const at = to.part + (long long)row * D + 8 * c8;
    *reinterpret_cast<f32x4*>(at) = a;
    *reinterpret_cast<f32x4*>(at + 4) = b;
    if (c8 == 0) {
      float* const stats = to.part + (long long)to.part_rows * D + row;
      stats[0] = M, stats[to.part_rows] = stats[2 * to.part_rows] = l;
    }
    return;
  }
  const int step = divide(r, job.by_group), head = r - step * job.G;
  const float nan = __uint_as_float(0x7FC00000u);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  typename Elem<T>::v8 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    out[e] = (T)(real ? (l == 0.f ? 0.f : a[e] * inv) : to.fill == 2 ? nan : 0.f);
    out[4 + e] = (T)(real ? (l == 0.f ? 0.f : b[e] * inv) : to.fill == 2 ? nan : 0.f);
  }
  *reinterpret_cast<typename Elem<T>::v8*>(static_cast<T*>(to.o) + step * to.o_step + head * to.o_head + 8 * c8) = out;
  if (c8 == 0 && to.lse)
    to.lse[step * to.l_step + head * to.l_head] =
        !real ? (to.fill == 2 ? nan : -INFINITY) : l == 0.f ? -INFINITY : fmaf(M, job.scale, log2f(l) * kLn2);
}

// Few rows.
template <class T, int kDH, bool kAligned, int kW>
__device__ __forceinline__ void run_few(const Source& src, const Job& job, const Sink& to, int D, unsigned char* lds,
                                        Stats<kW>& st) {
  constexpr int kBytes = 2 * kDH * kHalfBytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  unsigned char* const block = lds + wave * kBytes;
  const uint32_t block_at = tfgfa::lds_addr(block);
  const int count = max(0, (job.last - job.first - wave + kW - 1) / kW);
  auto key = [&](int n) { return (job.first + wave + n * kW) * kBlock; };
  State<T, kDH, 2> w;
  const float inv = 1.f / job.scale_log2;
  w.init(lane);
  Loader<kDH, kAligned, 2> in;
  typename Loader<kDH, kAligned, 2>::Place place = {};
  in.init(src, D, 0, lane);
  const int least = job.causal ? job.seen + divide(job.row0, job.by_group) + 1 : job.seen;
  auto pass = [&](auto exact) {
    if (count > 0) place = in.look_up(src, key(0));
    if (!decltype(exact)::value) load_rows(w, job, job.row0, D, lane);
#pragma unroll 1
    for (int n = 0; n < count; ++n) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the block before
      in.template issue<false>(src, key(n), place, block_at);
      in.template issue<true>(src, key(n), place, block_at + kBytes / 2);
      if (n + 1 < count) place = in.look_up(src, key(n + 1));
      tfgfa::wait_vmcnt<0>();
      w.template step<decltype(exact)::value>(block, block + kBytes / 2, key(n), least, job.scale_log2, inv, lane);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  pass(std::false_type());
  if (w.any_nan()) {
    w.clear();
    pass(std::true_type());
  }
  __syncthreads();  // (the rows' places are the blocks')
  w.publish(lds + wave * kBlock * 64 * kDH * 4, st.m + wave * kBlock, st.l + wave * kBlock, lane);
  __syncthreads();
  for (int e = tid; e < kBlock * 8 * kDH; e += 64 * kW)
    if (e % (8 * kDH) * 8 < D) put<T, kDH, kW>(lds, st, e / (8 * kDH), e % (8 * kDH), job, to, D);
}

// Many rows.  Two K tiles and two V tiles of 64 keys in LDS.  Step j of the workgroup: block 2j; wait for K of tile j + 1 and
// V of tile j, barrier, load V of tile j + 1 and K of tile j + 2; block 2j + 1.
template <class T, int kDH, bool kAligned, bool kLse>
__device__ __forceinline__ void run_many(const Source& src, const Job& job, const Sink& to, int D, unsigned char* lds) {
  constexpr int kHalf = kDH * kHalfBytes, kSlot = 2 * kHalf;  // K (or V) of a block, of a tile
  typedef State<T, kDH, 1> W;
  __shared__ int sh_again;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const uint32_t ring_at = tfgfa::lds_addr(lds);
  const int blocks = max(0, job.last - job.first), tiles = (blocks + 1) / 2;
  auto key = [&](int tile) { return job.first * kBlock + tile * kTile; };
  W w;
  const float c = job.scale_log2;
  w.init(lane);
  if (tid == 0) sh_again = 0;
  typedef Loader<kDH, kAligned, 1> In;                        // 16 keys of a tile: half a block
  In in;
  in.init(src, D, wave & 1, lane);
  const int mine = (wave >> 1) * kBlock;                      // the block's first key in the tile
  const int r0 = job.row0 + wave * kBlock, r1 = min(job.rows, r0 + kBlock) - 1;
  const int least = r0 >= job.rows ? 0 : job.causal ? job.seen + divide(r0, job.by_group) + 1 : job.seen;
  const int most = r0 >= job.rows ? 0 : job.causal ? job.seen + divide(r1, job.by_group) + 1 : job.seen;
  // Blocks with a key that some row of the wave sees, and those with none that one does not.
  const int act = min(blocks, max(0, (most + kBlock - 1) / kBlock - job.first));
  const int full = min(act, max(0, least / kBlock - job.first));
  auto issue = [&](auto value, int tile, const typename In::Place& place) {
    constexpr bool kValue = decltype(value)::value;
    in.template issue<kValue>(src, key(tile) + mine, place, ring_at + ((kValue ? 2 : 0) + (tile & 1)) * kSlot + (wave >> 1) * kHalf);
  };
  auto look_up = [&](int tile) { return in.look_up(src, key(tile) + mine); };
  const std::false_type keys{};
  const std::true_type values{};

  typename In::Place k_at = {}, v_at = {};
  if (tiles > 0) {
    v_at = look_up(0);
    issue(keys, 0, v_at);
    issue(values, 0, v_at);
  }
  if (tiles > 1) {
    v_at = look_up(1);
    issue(keys, 1, v_at);
  }
  if (tiles > 2) k_at = look_up(2);
  load_rows(w, job, r0, D, lane);
  tfgfa::wait_vmcnt<0>();
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  w.m = -INFINITY;
  const float head = fminf(Elem<T>::kHead, 1e30f * c);
  f32x16 s;
  typename W::v8 part[1][2];
  if (act > 0) w.scores(s, lds);
  // Half a step: block u, V of the one before it and K of the one after it in LDS.
  auto block = [&](int u, const unsigned char* v, const unsigned char* k, auto first) {
    if (u >= full) w.mask(s, (job.first + u) * kBlock, lane);
    w.template fused<!decltype(first)::value, kLse>(v, k, s, part, c, head);
  };
  auto last = [&](const unsigned char* v) { w.output(v, part); };
  auto turn = [&](int j) {  // between the halves of step j
    tfgfa::wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (j + 1 < tiles) issue(values, j + 1, v_at);
    if (j + 2 < tiles) issue(keys, j + 2, k_at);
    v_at = k_at;
    if (j + 3 < tiles) k_at = look_up(j + 3);
  };
  auto k_of = [&](int slot) { return lds + slot * kSlot; };
  auto v_of = [&](int slot) { return lds + (2 + slot) * kSlot; };
  // Steps both of whose blocks the wave computes: no branches, so that the accumulators stay where they are.
  auto step = [&](int j, auto slot, auto first) {
    constexpr int kS = decltype(slot)::value;
    block(2 * j, v_of(kS ^ 1) + kHalf, k_of(kS) + kHalf, first);
    turn(j);
    block(2 * j + 1, v_of(kS), k_of(kS ^ 1), std::false_type());
  };
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};
  const int steady = act / 2;
  int j = 0;
  if (steady > 0) {
    step(0, even, std::true_type());
#pragma unroll 1
    for (j = 1; j + 1 < steady; j += 2) {
      step(j, odd, std::false_type());
      step(j + 1, even, std::false_type());
    }
    if (j < steady) {
      step(j, odd, std::false_type());
      ++j;
    }
  }
  // The wave's last block alone, or what is left of the block before; then loads for the other waves.
  if (j < tiles) {
    const unsigned char* const v_last = v_of((j & 1) ^ 1) + kHalf;
    if (act & 1) {
      if (act == 1)
        block(0, v_last, k_of(0) + kHalf, std::true_type());
      else
        block(2 * j, v_last, k_of(j & 1) + kHalf, std::false_type());
    } else if (act > 0) {
      last(v_last);
    }
    turn(j);
    if (act & 1) last(v_of(j & 1));
    for (++j; j < tiles; ++j) turn(j);
  } else if (act > 0) {
    last(v_of((tiles - 1) & 1) + kHalf);
  }
  // The offset is c top - head rounded, weights are of c s exactly: the row's largest is 2^(head + what rounding left), at most
  // 2^(head + 1) below kFar, and from there on may be past the type on either side.  Offsets only rise, and what an earlier
  // one lost is 0 beside the last.  (kLowest, too, is what scores past float32's range in the log2 domain leave.)
  constexpr float kFar = 0x1p24f;
  const bool far = act > 0 && w.seen > job.first * kBlock && !(fabsf(w.m) < kFar);
  w.rescale(c);
  w.thr = 0.f;
  if ((__builtin_amdgcn_ballot_w64(far) != 0 || w.any_nan()) && lane == 0) sh_again = 1;
  __syncthreads();
  if (uniform(sh_again)) {
    // The exact pass: a tile at a time.
    const float inv = 1.f / c;
    w.clear();
#pragma unroll 1
    for (int n = 0; n < tiles; ++n) {
      const typename In::Place place = look_up(n);
      issue(keys, n, place);
      issue(values, n, place);
      tfgfa::wait_vmcnt<0>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll 1
      for (int b = 0; b < 2; ++b) {
        const int at = key(n) + b * kBlock;
        if (at < most && 2 * n + b < blocks)
          w.template step<true>(lds + (n & 1) * kSlot + b * kHalf, lds + (2 + (n & 1)) * kSlot + b * kHalf, at, least, c, inv, lane);
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
  }
  __syncthreads();
  // A row's dims are its two lanes': 4 of every 8 each.
  const int i = lane & 31, h = lane >> 5, row = wave * kBlock + i, r = job.row0 + row;
  const auto add = [](float x, float y) { return x + y; };
  const float l = over_pair(w.l, add), lp = over_pair(w.lp, add);
  const float m = w.thr == -INFINITY ? -INFINITY : w.m;
  const bool real = r < job.rows;
  if (to.part) {
    if (!real) return;
#pragma unroll
    for (int j = 0; j < 2 * kDH; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * j + 8 * g < D)
          *reinterpret_cast<f32x4*>(to.part + (long long)row * D + 32 * j + 8 * g + 4 * h) =
              f32x4{w.o[j][4 * g], w.o[j][4 * g + 1], w.o[j][4 * g + 2], w.o[j][4 * g + 3]};
    if (h == 0) {
      float* const stats = to.part + (long long)to.part_rows * D + row;
      stats[0] = m, stats[to.part_rows] = l, stats[2 * to.part_rows] = lp;
    }
    return;
  }
  typedef T v4 __attribute__((ext_vector_type(4)));
  const int step_of = divide(r, job.by_group), head_of = r - step_of * job.G;
  const bool stored = real || (to.fill != 0 && r < to.fill_to);
  const float nan = __uint_as_float(0x7FC00000u), inv = lp == 0.f ? 0.f : 1.f / lp;
  T* const out = static_cast<T*>(to.o) + step_of * to.o_step + head_of * to.o_head;
#pragma unroll
  for (int j = 0; j < 2 * kDH; ++j)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      uint32_t x[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = (T)(real ? (lp == 0.f ? 0.f : w.o[j][4 * (g + k) + e] * inv) : to.fill == 2 ? nan : 0.f);
        const auto two = __builtin_bit_cast(u32x2, y);
        x[k][0] = two[0], x[k][1] = two[1];
      }
      // The first lane takes dims 8 g .. of both, the second the next 8.
      const auto a = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
      const int d = 32 * j + 8 * (g + h);
      if (stored && d < D) *reinterpret_cast<u32x4*>(out + d) = u32x4{a[0], b[0], a[1], b[1]};
    }
  if (stored && h == 0 && to.lse)
    to.lse[step_of * to.l_step + head_of * to.l_head] =
        !real ? (to.fill == 2 ? nan : -INFINITY) : l == 0.f ? -INFINITY : fmaf(m, job.scale, log2f(l) * kLn2);
}

// ---------------------------------------------------------------------------------------
// Joining the parts of a job's rows: 16 lanes, 8 dims each, take every kSplit-th part of a row; kSplit such groups a row.

constexpr int kLanes = kMaxD / 8;
constexpr int kSplit = 4;
constexpr int kJoinRows = kThreads / kLanes / kSplit;  // rows of a workgroup
constexpr int kMine = kMaxParts / kLanes;  // parts whose statistics a lane has
constexpr int kAtOnce = kLanes / kSplit;   // parts whose sums a thread loads together

// A row's parts: `count` of them, `stride` floats apart, the sums of part 0 at `sums` (this lane's dims) and its offset at
// `stats` (the sums of weights `rows` and 2 `rows` further).
struct Parts {
  const float* sums;
  const float* stats;
  long long stride;
  int count, rows;
};
__device__ __forceinline__ Parts parts_of(const float* part, long long job, int count, int rows, int row, int D, int c8) {
  const long long stride = part_floats(rows, D);
  const float* const at = part + job * count * stride;
  return {at + (long long)row * D + 8 * c8, at + (long long)rows * D + row, stride, count, rows};
}

template <class F>
__device__ __forceinline__ float over_lanes(float x, F f) {
#pragma unroll
  for (int n = kLanes / 2; n > 0; n /= 2) x = f(x, __shfl_xor(x, n, kLanes));
  return x;
}

struct Joined {
  f32x4 a, b;
  float M, l, lp;
};

// The sum over kSources lists of parts, in the lanes of a row's first group; c: the lane in its group.  Every thread of the
// workgroup comes here.  (Dims past D: any that are there.)
template <int kSources>
__device__ __forceinline__ Joined join(const Parts (&from)[kSources], float scale_log2) {
  __shared__ f32x4 sh_sum[kThreads][2];
  const int tid = threadIdx.x, c = tid % kLanes, group = tid / kLanes % kSplit;
  Joined y = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.f, 0.f};
  float f[kSources][kMine], l[kSources][kMine], lp[kSources][kMine];
#pragma unroll
  for (int n = 0; n < kSources; ++n)
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int s = i * kLanes + c;
      const float* const at = from[n].stats + s * from[n].stride;
      const bool in = s < from[n].count;
      f[n][i] = in ? at[0] : -INFINITY;
      l[n][i] = in ? at[from[n].rows] : 0.f;
      lp[n][i] = in ? at[2 * from[n].rows] : 0.f;
      y.M = fmaxf(y.M, f[n][i]);
    }
  y.M = over_lanes(y.M, [](float u, float v) { return fmaxf(u, v); });
#pragma unroll
  for (int n = 0; n < kSources; ++n)
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      f[n][i] = f[n][i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((f[n][i] - y.M) * scale_log2);
      y.l = fmaf(f[n][i], l[n][i], y.l), y.lp = fmaf(f[n][i], lp[n][i], y.lp);
    }
  y.l = over_lanes(y.l, [](float u, float v) { return u + v; });
  y.lp = over_lanes(y.lp, [](float u, float v) { return u + v; });
#pragma unroll
  for (int n = 0; n < kSources; ++n)
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int here = min(kLanes, from[n].count - i * kLanes);
      const float* const first = from[n].sums + i * kLanes * from[n].stride;
      if (here <= 0) continue;
      f32x4 u[kAtOnce], v[kAtOnce];
      float w[kAtOnce];
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s) {
        const int at = s * kSplit + group;
        const float* const row = first + min(at, here - 1) * from[n].stride;
        u[s] = *reinterpret_cast<const f32x4*>(row), v[s] = *reinterpret_cast<const f32x4*>(row + 4);
        w[s] = __shfl(f[n][i], at, kLanes);  // (past `here` there is a weight of 0: no part)
      }
#pragma unroll
      for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y.a[e] = w[s] == 0.f ? y.a[e] : fmaf(w[s], u[s][e], y.a[e]);
          y.b[e] = w[s] == 0.f ? y.b[e] : fmaf(w[s], v[s][e], y.b[e]);
        }
    }
  sh_sum[tid][0] = y.a, sh_sum[tid][1] = y.b;
  __syncthreads();
  if (group == 0)
#pragma unroll
    for (int g = 1; g < kSplit; ++g) y.a += sh_sum[tid + g * kLanes][0], y.b += sh_sum[tid + g * kLanes][1];
  return y;
}

template <class T>
__device__ __forceinline__ void store_row(T* to, const Joined& y, bool zero, bool nan) {
  const float inv = y.lp == 0.f ? 0.f : 1.f / y.lp, bad = __uint_as_float(0x7FC00000u);
  typename Elem<T>::v8 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    out[e] = (T)(nan ? bad : zero || y.lp == 0.f ? 0.f : y.a[e] * inv);
    out[4 + e] = (T)(nan ? bad : zero || y.lp == 0.f ? 0.f : y.b[e] * inv);
  }
  *reinterpret_cast<typename Elem<T>::v8*>(to) = out;
}
__device__ __forceinline__ float row_lse(const Joined& y, float scale, bool zero, bool nan) {
  return nan ? __uint_as_float(0x7FC00000u) : zero || y.l == 0.f ? -INFINITY : fmaf(y.M, scale, log2f(y.l) * kLn2);
}

// ---------------------------------------------------------------------------------------
// New tokens of each sequence.

struct AttendArgs {
  const void* q;
  void* o;
  float* lse;
  float* part;
  const char* k;
  const char* v;
  Pages ks, vs;
  Rows qs, os;
  const int* table;
  long long table_stride;
  const int* lens;
  const int* lengths;
  Division by_page, by_group;
  int page, P, n_max, N, G, Hkv, heads, D, causal, pad, tiles, parts, part_rows;
  float scale, scale_log2;
};

// How many rows a workgroup takes, and how.
enum class Kind { kFew, kFewWide, kMany };
__host__ __device__ constexpr int rows_of(Kind kind) {
  return kind == Kind::kMany ? kManyRows : kBlock;
}
constexpr int waves_of(Kind kind) { return kind == Kind::kFewWide ? 8 : kWaves; }
constexpr int lds_of(Kind kind, int kDH) { return kind == Kind::kMany ? many_lds(kDH) : few_lds(kDH, waves_of(kind)); }

// Waves a SIMD, which bound the registers.  Many rows, heads of 64: 3 (8192 causal tokens of 16 heads 178 us, with 2 188; 151 to
// 157 since, by its steps without branches); few rows: 4, which their registers leave anyhow (64 sequences on 4 prefixes 27 us
// with a bound of 4 and of 2).
constexpr int simd_waves(Kind kind, int kDH) {
  return kDH == 2 ? 2 : kind == Kind::kMany ? 3 : 4;
}

template <class T, int kDH, bool kAligned, Kind kKind, bool kLse>
__device__ __forceinline__ void run(const Source& src, const Job& job, const Sink& to, int D, unsigned char* lds,
                                    Stats<waves_of(kKind)>& st) {
  if constexpr (kKind == Kind::kMany)
    run_many<T, kDH, kAligned, kLse>(src, job, to, D, lds);
  else
    run_few<T, kDH, kAligned, waves_of(kKind)>(src, job, to, D, lds, st);
}

// Which head, part and tile of rows a workgroup takes; in either order the workgroups of a head are on one XCD where 8 divides
// the heads.
struct Work {
  int head, part, tile;
};
// Tile after tile.
__device__ __forceinline__ Work by_tiles(int idx, int heads, int parts) {
  const int rest = idx / heads, tile = rest / parts;
  return {idx - rest * heads, rest - tile * parts, tile};
}
// The tiles of a part together, 8 parts at a time, so that its keys come from HBM once.
__device__ __forceinline__ Work by_heads(int idx, int heads, int parts, int tiles) {
  const int first = idx / (8 * tiles), in = idx - first * 8 * tiles, width = min(8, heads * parts - 8 * first);
  const int tile = in / width, job = 8 * first + in - tile * width, part = job / heads;
  return {job - part * heads, part, tile};
}

// Part s of S of `blocks` blocks: whole rounds of the workgroup.
template <Kind kKind>
__device__ __forceinline__ void share(Job* job, int blocks, int s, int S) {
  constexpr int kRound = kKind == Kind::kMany ? 2 : waves_of(kKind);
  const int rounds = (blocks + kRound - 1) / kRound;
  job->first = kRound * (int)((long long)rounds * s / S);
  job->last = min(blocks, kRound * (int)((long long)rounds * (s + 1) / S));
}

template <class T, int kDH, bool kAligned, Kind kKind, bool kLse>
__global__ __launch_bounds__(64 * waves_of(kKind), simd_waves(kKind, kDH)) void attend_kernel(const AttendArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[lds_of(kKind, kDH)];
  __shared__ Stats<waves_of(kKind)> st;
  constexpr int kRows = rows_of(kKind);
  // The longest first (the last tiles of a causal sequence); a key-value head's workgroups on one XCD where 8 divides
  // their number.
  const bool together = kKind != Kind::kMany && a.tiles > 1;
  const Work at = together ? by_heads(blockIdx.x, a.heads, a.parts, a.tiles) : by_tiles(blockIdx.x, a.heads, a.parts);
  const int head = at.head, s = at.part, tile = a.tiles - 1 - at.tile;
  const int b = head / a.Hkv, kv = head - b * a.Hkv;
  const int len = ((uniform_ints)a.lens)[b], n = a.lengths ? ((uniform_ints)a.lengths)[b] : a.N;
  const bool fits = len >= 0 && n >= 0 && n <= a.N && (long long)len + (a.causal ? n : 0) <= a.n_max;
  const long long first_head = (long long)kv * a.G;
  Job job;
  job.q = static_cast<const T*>(a.q) + b * a.qs.b + first_head * a.qs.h;
  job.q_step = a.qs.n, job.q_head = a.qs.h;
  job.by_group = a.by_group, job.G = a.G, job.row0 = tile * kRows, job.rows = fits ? n * a.G : 0;
  job.seen = fits ? len : 0, job.causal = a.causal;
  job.scale = a.scale, job.scale_log2 = a.scale_log2;
  const int top = min(job.rows, job.row0 + kRows) - 1;
  const int keys = job.row0 >= job.rows ? 0 : a.causal ? len + divide(top, a.by_group) + 1 : len;
  share<kKind>(&job, (keys + kBlock - 1) / kBlock, s, a.parts);
  const Source src = {a.k + kv * a.ks.h, a.v + kv * a.vs.h, a.ks, a.vs, a.table + b * a.table_stride, a.by_page, a.page, a.P, keys};
  const long long unit = (long long)head * a.tiles + tile;
  Sink to;
  to.o = static_cast<T*>(a.o) + b * a.os.b + first_head * a.os.h;
  to.o_step = a.os.n, to.o_head = a.os.h;
  to.lse = a.lse ? a.lse + ((long long)b * a.Hkv * a.G + first_head) * a.N : nullptr;
  to.l_step = 1, to.l_head = a.N;
  to.part = a.parts > 1 ? a.part + (unit * a.parts + s) * part_floats(a.part_rows, a.D) : nullptr;
  to.part_rows = a.part_rows;
  to.fill_to = a.N * a.G, to.fill = !fits ? 2 : a.pad;
  run<T, kDH, kAligned, kKind, kLse>(src, job, to, a.D, lds, st);
}

template <class T, Kind kKind>
__global__ __launch_bounds__(kThreads) void attend_join_kernel(const AttendArgs a) {
  constexpr int kRows = rows_of(kKind), kBlocks = kRows / kJoinRows;
  const int c = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int unit = blockIdx.x / kBlocks, row = (int)(blockIdx.x % kBlocks) * kJoinRows + group / kSplit;
  const int head = unit / a.tiles, tile = unit - head * a.tiles, b = head / a.Hkv, kv = head - b * a.Hkv;
  const int r = tile * kRows + row, step = divide(r, a.by_group), h = kv * a.G + r - step * a.G;
  const int len = a.lens[b], n = a.lengths ? a.lengths[b] : a.N;
  const bool fits = len >= 0 && n >= 0 && n <= a.N && (long long)len + (a.causal ? n : 0) <= a.n_max;
  const bool past = fits && step >= n;
  const int d = 8 * c < a.D ? c : 0;
  Parts p[1] = {parts_of(a.part, unit, a.parts, a.part_rows, row, a.D, d)};
  if (!fits || step >= n) p[0].count = 0;
  const Joined y = join(p, a.scale_log2);
  if (group % kSplit != 0 || step >= a.N || (past && !a.pad)) return;
  if (8 * c < a.D) store_row(static_cast<T*>(a.o) + b * a.os.b + h * a.os.h + step * a.os.n + 8 * c, y, past, !fits);
  if (c == 0 && a.lse) a.lse[((long long)b * a.Hkv * a.G + h) * a.N + step] = row_lse(y, a.scale, past, !fits);
}

// ---------------------------------------------------------------------------------------
// A decode step of sequences that share a prefix.

struct SharedArgs {
  const void* q;
  void* o;
  float* lse;
  float* prefix_part;
  float* own_part;
  char* k;
  char* v;
  const void* kn;
  const void* vn;
  Pages ks, vs;
  Vecs qs, os, kns, vns;
  const int* prefix_table;
  const int* prefix_lens;
  const int* table;
  const int* lens;
  long long prefix_stride, table_stride;
  Division by_page, by_group;
  int page, P, prefix_max, n_max, G, Hkv, R, each, D;   // each: sequences of a group
  int prefix_heads, prefix_tiles, prefix_parts, prefix_part_rows, prefix_jobs;
  int own_heads, own_tiles, own_parts, own_part_rows;
  float scale, scale_log2;
};

template <class T, int kDH, bool kAligned, Kind kKind>
__global__ __launch_bounds__(64 * waves_of(kKind), simd_waves(kKind, kDH)) void shared_kernel(const SharedArgs a) {
  constexpr int kPrefixLds = lds_of(kKind, kDH), kOwnLds = lds_of(Kind::kFew, kDH);
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kPrefixLds > kOwnLds ? kPrefixLds : kOwnLds];
  __shared__ Stats<waves_of(kKind)> st;
  Job job;
  Sink to;
  job.by_group = a.by_group, job.G = a.G, job.causal = 0;
  job.q_step = a.qs.b, job.q_head = a.qs.h;
  job.scale = a.scale, job.scale_log2 = a.scale_log2;
  to.o = nullptr, to.o_step = to.o_head = 0, to.lse = nullptr, to.l_step = to.l_head = 0, to.fill_to = to.fill = 0;
  const bool prefix = (int)blockIdx.x < a.prefix_jobs;
  const int idx = prefix ? blockIdx.x : blockIdx.x - a.prefix_jobs;
  const int heads = prefix ? a.prefix_heads : a.own_heads, parts = prefix ? a.prefix_parts : a.own_parts;
  const int tiles = prefix ? a.prefix_tiles : a.own_tiles;
  const bool together = tiles > 1 && !(prefix && kKind == Kind::kMany);
  const Work at = together ? by_heads(idx, heads, parts, tiles) : by_tiles(idx, heads, parts);
  const int head = at.head, tile = at.tile, s = at.part;
  const int b = head / a.Hkv, kv = head - b * a.Hkv;   // group or sequence
  Source src = {a.k + kv * a.ks.h, a.v + kv * a.vs.h, a.ks, a.vs, nullptr, a.by_page, a.page, a.P, 0};
  const long long first_head = (long long)kv * a.G;
  if (prefix) {
    constexpr int kRows = rows_of(kKind);
    const int len = ((uniform_ints)a.prefix_lens)[b];
    src.table = a.prefix_table + b * a.prefix_stride;
    src.keys = len >= 0 && len <= a.prefix_max ? len : 0;
    job.q = static_cast<const T*>(a.q) + (long long)b * a.each * a.qs.b + first_head * a.qs.h;
    job.row0 = tile * kRows, job.rows = a.each * a.G, job.seen = src.keys;
    share<kKind>(&job, (src.keys + kBlock - 1) / kBlock, s, parts);
    to.part_rows = a.prefix_part_rows;
    to.part = a.prefix_part + (((long long)head * a.prefix_tiles + tile) * parts + s) * part_floats(a.prefix_part_rows, a.D);
    run<T, kDH, kAligned, kKind, true>(src, job, to, a.D, lds, st);
  } else {
    constexpr int kRows = rows_of(Kind::kFew);
    const int append = a.kn != nullptr, len = ((uniform_ints)a.lens)[b];
    const bool fits = len >= 0 && len <= a.n_max - append;
    src.table = a.table + b * a.table_stride;
    src.keys = fits ? len + append : 0;
    // The new row goes to its page first; this workgroup alone reads it (or another with rows of the same head, which
    // writes the same bytes before it reads them).
    if (append && fits && s == parts - 1) {
      const int at = divide(len, a.by_page), id = ((uniform_ints)src.table)[at], tid = threadIdx.x;
      const bool value = tid >= kMaxD / 8;
      const int c = value ? tid - kMaxD / 8 : tid;
      if ((uint32_t)id < (uint32_t)a.P && 8 * c < a.D && tid < kMaxD / 4) {
        const Pages& ps = value ? a.vs : a.ks;
        const T* const from = value ? static_cast<const T*>(a.vn) + b * a.vns.b + kv * a.vns.h
                                    : static_cast<const T*>(a.kn) + b * a.kns.b + kv * a.kns.h;
        char* const row = (value ? a.v : a.k) + kv * ps.h + (uint64_t)(uint32_t)id * (uint64_t)ps.p + (uint64_t)(len - at * a.page) * (uint64_t)ps.n;
        *reinterpret_cast<u32x4*>(row + 16 * c) = *reinterpret_cast<const u32x4*>(from + 8 * c);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    job.q = static_cast<const T*>(a.q) + b * a.qs.b + first_head * a.qs.h;
    job.row0 = tile * kRows, job.rows = a.G, job.seen = src.keys;
    share<Kind::kFew>(&job, (src.keys + kBlock - 1) / kBlock, s, parts);
    to.part_rows = a.own_part_rows;
    to.part = a.own_part + (((long long)head * a.own_tiles + tile) * parts + s) * part_floats(a.own_part_rows, a.D);
    run<T, kDH, kAligned, Kind::kFew, true>(src, job, to, a.D, lds, st);
  }
}

template <class T, Kind kKind>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(const SharedArgs a, int rows) {
  constexpr int kRows = rows_of(kKind);
  const int c = threadIdx.x % kLanes, group = threadIdx.x / kLanes, mine = blockIdx.x * kJoinRows + group / kSplit;
  const int at = min(mine, rows - 1);
  const int H = a.Hkv * a.G, b = at / H, h = at - b * H, kv = h / a.G, g = h - kv * a.G, r = b / a.each;
  const int plen = a.prefix_lens[r], len = a.lens[b];
  const bool fits = plen >= 0 && plen <= a.prefix_max && len >= 0 && len <= a.n_max - (a.kn ? 1 : 0);
  const int d = 8 * c < a.D ? c : 0;
  const int row = (b - r * a.each) * a.G + g;
  Parts p[2] = {
      parts_of(a.prefix_part, ((long long)r * a.Hkv + kv) * a.prefix_tiles + row / kRows, a.prefix_parts, a.prefix_part_rows,
               row % kRows, a.D, d),
      parts_of(a.own_part, ((long long)b * a.Hkv + kv) * a.own_tiles + g / kBlock, a.own_parts, a.own_part_rows, g % kBlock, a.D, d)};
  const Joined y = join(p, a.scale_log2);
  if (group % kSplit != 0 || mine >= rows) return;
  if (8 * c < a.D) store_row(static_cast<T*>(a.o) + b * a.os.b + h * a.os.h + 8 * c, y, false, !fits);
  if (c == 0 && a.lse) a.lse[at] = row_lse(y, a.scale, false, !fits);
}

// ---------------------------------------------------------------------------------------
// Host side.

constexpr int kCu = 256;  // workgroups are counted for this many CUs, so that a workspace's size does not depend on the device

constexpr long long kMaxGroups = UINT32_MAX / kThreads;  // workgroups of a launch: fewer than 2^32 threads

// 33 to 64 rows: 40 tokens of 8 sequences, 25 heads, take 14.7 us as two tiles of few and 19.5 as a tile of many, two thirds empty;
// 8 prefixes for 16 sequences each, heads of 128, 43.3 and 38.2, but then with weights rounded once.  65 to 128: 32 tokens of 32 sequences, 32 heads
// on 8 of 128, take 69 as many and 101 as few, 100 tokens of 8 sequences 21.7 and 18.5.
static Kind choose_kind(long long rows) {
  return rows <= 2 * kBlock ? Kind::kFew : Kind::kMany;
}
// Workgroups that a job of up to n_max keys is divided over, where there are `jobs` of them: `slots` a CU in all, parts of at
// least `least` keys.
static int choose_parts(long long slots, long long jobs, long long n_max, long long least) {
  const long long parts = std::min({slots * kCu / std::max(1LL, jobs), n_max / least, (long long)kMaxParts});
  return (int)std::max(1LL, parts);
}
// Rows that a part keeps of a job of `rows`: those of its largest tile.
static int part_rows(Kind kind, long long rows) { return (int)std::min<long long>(rows_of(kind), rows); }
static size_t part_bytes(int rows, long long jobs, int parts, int D) {
  return ((size_t)jobs * parts * part_floats(rows, D) * 4 + 255) / 256 * 256;
}

static bool heads_ok(int B, int H, int Hkv, int page, int M) {
  if (B < 0 || H < 0 || Hkv < 0 || page < 1 || M < 0) return false;
  return Hkv == 0 ? H == 0 : H % Hkv == 0;
}

struct AttendPlan {
  Kind kind;
  long long tiles, jobs;
  int parts, part_rows;
  size_t bytes;
};
// False: too large.
static bool attend_plan(int B, int H, int Hkv, int N, int page, int M, int D, AttendPlan* x) {
  const long long n_max = (long long)M * page, rows = (long long)N * (H / Hkv);
  if (n_max > INT32_MAX - (1 << 20) || rows > INT32_MAX - kManyRows || (long long)B * Hkv > INT32_MAX) return false;
  x->kind = choose_kind(rows);
  const int each = rows_of(x->kind);
  x->tiles = (rows + each - 1) / each;
  if (x->tiles > INT32_MAX / ((long long)B * Hkv)) return false;
  x->jobs = x->tiles * B * Hkv;
  // Eight waves a workgroup where a CU has one (12 tokens of 8 sequences, 32 heads on 8 of 128, 14.6 us, with four 18.5; 4
  // tokens behind 1020, 8 times, 25 heads, 11.8 and 13.7; 2 behind 500, 64 times, 12 heads, 18.1 and 14.8, so not there).
  if (x->kind == Kind::kFew && x->jobs <= kCu) x->kind = Kind::kFewWide;
  // Two workgroups a CU, parts of 256 keys or more (512 tokens behind 16000, 32 heads on 8 of 128: 142 us, with one 157, with
  // three 150).  Fewer than four parts of a short cache cost more in joining than they gain (4 tokens behind 1020, 8 times, 25
  // heads: 13.7 us whole, 16.7 in two, of four waves).
  x->parts = choose_parts(x->kind == Kind::kFewWide ? 1 : 2, x->jobs, n_max, 256);
  if (x->parts < 4 && n_max < 4096) x->parts = 1;
  x->part_rows = part_rows(x->kind, rows);
  x->bytes = x->parts > 1 ? part_bytes(x->part_rows, x->jobs, x->parts, D) : 0;
  return x->jobs * x->parts <= kMaxGroups;  // (the join has at most kManyRows / kJoinRows a job, of few jobs)
}

template <class T, int kDH, bool kAligned>
static void launch_attend(const AttendArgs& a, const AttendPlan& x, hipStream_t stream) {
  const dim3 grid((unsigned)(x.jobs * x.parts));
  if (x.kind == Kind::kFewWide)
    hipLaunchKernelGGL((attend_kernel<T, kDH, kAligned, Kind::kFewWide, true>), grid, dim3(64 * waves_of(Kind::kFewWide)), 0,
                       stream, a);
  else if (x.kind == Kind::kFew)
    hipLaunchKernelGGL((attend_kernel<T, kDH, kAligned, Kind::kFew, true>), grid, dim3(kThreads), 0, stream, a);
  else if (a.lse)
    hipLaunchKernelGGL((attend_kernel<T, kDH, kAligned, Kind::kMany, true>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((attend_kernel<T, kDH, kAligned, Kind::kMany, false>), grid, dim3(kThreads), 0, stream, a);
}
template <class T>
static hipError_t launch_attend(const AttendArgs& a, const AttendPlan& x, hipStream_t stream) {
  const bool aligned = a.page % kGroup == 0;
  if (a.D <= 64)
    aligned ? launch_attend<T, 1, true>(a, x, stream) : launch_attend<T, 1, false>(a, x, stream);
  else
    aligned ? launch_attend<T, 2, true>(a, x, stream) : launch_attend<T, 2, false>(a, x, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || x.parts == 1) return e;
  const dim3 grid((unsigned)(x.jobs * (rows_of(x.kind) / kJoinRows)));
  if (x.kind != Kind::kMany)
    hipLaunchKernelGGL((attend_join_kernel<T, Kind::kFew>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((attend_join_kernel<T, Kind::kMany>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

struct SharedPlan {
  Kind kind;
  long long prefix_tiles, prefix_jobs, own_tiles, own_jobs;  // jobs: without their parts
  int prefix_parts, prefix_part_rows, own_parts, own_part_rows;
  size_t own_at, bytes;
};
static bool shared_plan(int R, int B, int H, int Hkv, int page, int Mp, int M, int D, SharedPlan* x) {
  const long long n_max = (long long)M * page, p_max = (long long)Mp * page, G = H / Hkv, rows = B / R * G;
  if (n_max > INT32_MAX - (1 << 20) || p_max > INT32_MAX - (1 << 20) || rows > INT32_MAX - kManyRows)
    return false;
  x->kind = choose_kind(rows);
  x->prefix_tiles = (rows + rows_of(x->kind) - 1) / rows_of(x->kind);
  x->own_tiles = (G + kBlock - 1) / kBlock;
  x->prefix_jobs = x->prefix_tiles * R * Hkv;
  x->own_jobs = x->own_tiles * B * Hkv;
  // Few rows: two workgroups a CU for prefixes (2 of 30000 for 16 sequences each 59 us, with one 65; 1 of 8000 24, with one
  // 20), many: one, with the sequences' own beside them (1 of 32000 for 64 sequences 70, with two 76).
  x->prefix_parts = choose_parts(x->kind == Kind::kFew ? 2 : 1, x->prefix_jobs, p_max, x->kind == Kind::kMany ? 512 : 128);
  x->own_parts = choose_parts(2, x->own_jobs, n_max, 128);
  x->prefix_part_rows = part_rows(x->kind, rows), x->own_part_rows = part_rows(Kind::kFew, G);
  x->own_at = part_bytes(x->prefix_part_rows, x->prefix_jobs, x->prefix_parts, D);
  x->bytes = x->own_at + part_bytes(x->own_part_rows, x->own_jobs, x->own_parts, D);
  return x->prefix_jobs * x->prefix_parts + x->own_jobs * x->own_parts <= kMaxGroups && (long long)B * H <= kMaxGroups * kJoinRows;
}

template <class T, int kDH, bool kAligned>
static void launch_shared(const SharedArgs& a, const SharedPlan& x, hipStream_t stream) {
  const dim3 grid((unsigned)(x.prefix_jobs * x.prefix_parts + x.own_jobs * x.own_parts));
  if (x.kind == Kind::kFew)
    hipLaunchKernelGGL((shared_kernel<T, kDH, kAligned, Kind::kFew>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((shared_kernel<T, kDH, kAligned, Kind::kMany>), grid, dim3(kThreads), 0, stream, a);
}
template <class T>
static hipError_t launch_shared(const SharedArgs& a, const SharedPlan& x, int rows, hipStream_t stream) {
  const bool aligned = a.page % kGroup == 0;
  if (a.D <= 64)
    aligned ? launch_shared<T, 1, true>(a, x, stream) : launch_shared<T, 1, false>(a, x, stream);
  else
    aligned ? launch_shared<T, 2, true>(a, x, stream) : launch_shared<T, 2, false>(a, x, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((rows + kJoinRows - 1) / kJoinRows);
  if (x.kind == Kind::kFew)
    hipLaunchKernelGGL((shared_join_kernel<T, Kind::kFew>), grid, dim3(kThreads), 0, stream, a, rows);
  else
    hipLaunchKernelGGL((shared_join_kernel<T, Kind::kMany>), grid, dim3(kThreads), 0, stream, a, rows);
  return hipGetLastError();
}

// A pool's rows of a transfer are one buffer of less than 2^30 bytes.
static bool rows_fit(const Pages& st) { return st.n < (1 << 30) / kGroup; }

}  // namespace tfgfa_context

extern "C" size_t tfpages_attend_workspace(int B, int H, int H_kv, int N, int page, int M, int D) {
  using namespace tfgfa_context;
  if (!heads_ok(B, H, H_kv, page, M) || N < 0 || D < 8 || D > kMaxD || (D & 7)) return 0;
  if (B == 0 || H == 0 || N == 0) return 0;
  AttendPlan x;
  return attend_plan(B, H, H_kv, N, page, M, D, &x) ? x.bytes : 0;
}

extern "C" int tfpages_attend(const void* q, const int64_t* q_strides, const void* k_pages, const int64_t* k_strides,
                              const void* v_pages, const int64_t* v_strides, const int* page_table,
                              int64_t table_stride, const int* cache_seqlens, const int* lengths, void* o,
                              const int64_t* o_strides, float* lse, int pad, int causal, int B, int H, int H_kv,
                              int N, int P, int page, int M, int D, int dtype, float softmax_scale, void* workspace,
                              size_t workspace_bytes, void* hip_stream) {
  using namespace tfgfa_context;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16) return TFGFA_ERR_DTYPE;
  if (!heads_ok(B, H, H_kv, page, M) || N < 0 || P < 0) return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7)) return TFGFA_ERR_HEAD_DIM;
  if (!(softmax_scale > 0.f) || !isfinite(softmax_scale * kLog2e)) return TFGFA_ERR_SCALE;
  if (causal != 0 && causal != 1) return TFGFA_ERR_CAUSAL_FLAG;
  if (B == 0 || H == 0 || N == 0) return TFGFA_OK;
  if (P == 0) return TFGFA_ERR_BAD_SHAPE;
  AttendPlan x;
  if (!attend_plan(B, H, H_kv, N, page, M, D, &x)) return TFGFA_ERR_TOO_LARGE;
  if (!q || !k_pages || !v_pages || !o || !cache_seqlens || (!page_table && M > 0) || !q_strides || !k_strides ||
      !v_strides || !o_strides)
    return TFGFA_ERR_NULL_POINTER;
  AttendArgs a = {};
  if (!tfgfa::rows_ok(q_strides, B, H, N, D, &a.qs) || !tfgfa::rows_ok(o_strides, B, H, N, D, &a.os) ||
      !tfgfa::pages_ok(k_strides, P, H_kv, page, D, &a.ks) || !tfgfa::pages_ok(v_strides, P, H_kv, page, D, &a.vs) ||
      !tfgfa::pages_apart({2 * a.os.b, 2 * a.os.h, 2 * a.os.n}, B, H, N, D))
    return TFGFA_ERR_STRIDE;
  if (B > 1 && table_stride < 0) return TFGFA_ERR_STRIDE;
  if (!rows_fit(a.ks) || !rows_fit(a.vs)) return TFGFA_ERR_TOO_LARGE;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o | (uintptr_t)workspace) & 15u)
    return TFGFA_ERR_ALIGNMENT;
  if (((uintptr_t)page_table | (uintptr_t)cache_seqlens | (uintptr_t)lengths | (uintptr_t)lse) & 3u) return TFGFA_ERR_ALIGNMENT;
  if (x.bytes > (workspace ? workspace_bytes : 0)) x.parts = 1;
  a.q = q, a.o = o, a.lse = lse, a.part = static_cast<float*>(workspace);
  a.k = static_cast<const char*>(k_pages), a.v = static_cast<const char*>(v_pages);
  a.table = page_table, a.table_stride = B > 1 ? table_stride : 0, a.lens = cache_seqlens, a.lengths = lengths;
  a.by_page = tfgfa::division_by(page), a.by_group = tfgfa::division_by(H / H_kv);
  a.page = page, a.P = P, a.n_max = M * page, a.N = N, a.G = H / H_kv, a.Hkv = H_kv, a.heads = B * H_kv, a.D = D;
  a.causal = causal, a.pad = pad != 0, a.tiles = (int)x.tiles, a.parts = x.parts, a.part_rows = x.part_rows;
  a.scale = softmax_scale, a.scale_log2 = softmax_scale * kLog2e;
  const hipStream_t stream = (hipStream_t)hip_stream;
  const hipError_t e = dtype == TFGFA_DTYPE_BF16 ? launch_attend<__bf16>(a, x, stream) : launch_attend<_Float16>(a, x, stream);
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}

extern "C" size_t tfpages_decode_shared_workspace(int R, int B, int H, int H_kv, int page, int M_prefix, int M, int D) {
  using namespace tfgfa_context;
  if (!heads_ok(B, H, H_kv, page, M) || M_prefix < 0 || D < 8 || D > kMaxD || (D & 7) || R < 1 || B % R) return 0;
  if (B == 0 || H == 0) return 0;
  SharedPlan x;
  return shared_plan(R, B, H, H_kv, page, M_prefix, M, D, &x) ? x.bytes : 0;
}

extern "C" int tfpages_decode_shared(const void* q, const int64_t* q_strides, void* k_pages, const int64_t* k_strides,
                                     void* v_pages, const int64_t* v_strides, const int* prefix_table,
                                     int64_t prefix_stride, const int* prefix_lens, const int* page_table,
                                     int64_t table_stride, const int* cache_seqlens, const void* k_new,
                                     const int64_t* k_new_strides, const void* v_new, const int64_t* v_new_strides,
                                     void* o, const int64_t* o_strides, float* lse, int R, int B, int H, int H_kv,
                                     int P, int page, int M_prefix, int M, int D, int dtype, float softmax_scale,
                                     void* workspace, size_t workspace_bytes, void* hip_stream) {
  using namespace tfgfa_context;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16) return TFGFA_ERR_DTYPE;
  if (!heads_ok(B, H, H_kv, page, M) || M_prefix < 0 || P < 0 || R < 0 || (R == 0 ? B != 0 : B % R != 0))
    return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7)) return TFGFA_ERR_HEAD_DIM;
  if (!(softmax_scale > 0.f) || !isfinite(softmax_scale * kLog2e)) return TFGFA_ERR_SCALE;
  if ((k_new == nullptr) != (v_new == nullptr)) return TFGFA_ERR_NULL_POINTER;
  if (B == 0 || H == 0) return TFGFA_OK;
  if (P == 0) return TFGFA_ERR_BAD_SHAPE;
  SharedPlan x;
  if (!shared_plan(R, B, H, H_kv, page, M_prefix, M, D, &x)) return TFGFA_ERR_TOO_LARGE;
  if (!q || !k_pages || !v_pages || !o || !prefix_lens || !cache_seqlens || (!page_table && M > 0) ||
      (!prefix_table && M_prefix > 0) || !q_strides || !k_strides || !v_strides || !o_strides ||
      (k_new && (!k_new_strides || !v_new_strides)))
    return TFGFA_ERR_NULL_POINTER;
  SharedArgs a = {};
  if (!tfgfa::vecs_ok(q_strides, B, H, &a.qs) || !tfgfa::vecs_ok(o_strides, B, H, &a.os) ||
      !tfgfa::pages_ok(k_strides, P, H_kv, page, D, &a.ks) || !tfgfa::pages_ok(v_strides, P, H_kv, page, D, &a.vs) ||
      !tfgfa::apart(a.os.b, B, a.os.h, H, D))
    return TFGFA_ERR_STRIDE;
  if (k_new && (!tfgfa::vecs_ok(k_new_strides, B, H_kv, &a.kns) || !tfgfa::vecs_ok(v_new_strides, B, H_kv, &a.vns) ||
                !tfgfa::pages_apart(a.ks, P, H_kv, page, D) || !tfgfa::pages_apart(a.vs, P, H_kv, page, D)))
    return TFGFA_ERR_STRIDE;
  if ((B > 1 && table_stride < 0) || (R > 1 && prefix_stride < 0)) return TFGFA_ERR_STRIDE;
  if (!rows_fit(a.ks) || !rows_fit(a.vs)) return TFGFA_ERR_TOO_LARGE;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o | (uintptr_t)k_new | (uintptr_t)v_new |
       (uintptr_t)workspace) & 15u)
    return TFGFA_ERR_ALIGNMENT;
  if (((uintptr_t)prefix_table | (uintptr_t)prefix_lens | (uintptr_t)page_table | (uintptr_t)cache_seqlens |
       (uintptr_t)lse) & 3u)
    return TFGFA_ERR_ALIGNMENT;
  if (x.bytes > (workspace ? workspace_bytes : 0)) return TFGFA_ERR_SCRATCH;
  a.q = q, a.o = o, a.lse = lse;
  a.prefix_part = static_cast<float*>(workspace);
  a.own_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + x.own_at);
  a.k = static_cast<char*>(k_pages), a.v = static_cast<char*>(v_pages), a.kn = k_new, a.vn = v_new;
  a.prefix_table = prefix_table, a.prefix_lens = prefix_lens, a.table = page_table, a.lens = cache_seqlens;
  a.prefix_stride = R > 1 ? prefix_stride : 0, a.table_stride = B > 1 ? table_stride : 0;
  a.by_page = tfgfa::division_by(page), a.by_group = tfgfa::division_by(H / H_kv);
  a.page = page, a.P = P, a.prefix_max = M_prefix * page, a.n_max = M * page, a.G = H / H_kv, a.Hkv = H_kv, a.R = R;
  a.each = B / R, a.D = D;
  a.prefix_heads = R * H_kv, a.prefix_tiles = (int)x.prefix_tiles, a.prefix_parts = x.prefix_parts;
  a.prefix_part_rows = x.prefix_part_rows, a.prefix_jobs = (int)(x.prefix_jobs * x.prefix_parts);
  a.own_heads = B * H_kv, a.own_tiles = (int)x.own_tiles, a.own_parts = x.own_parts, a.own_part_rows = x.own_part_rows;
  a.scale = softmax_scale, a.scale_log2 = softmax_scale * kLog2e;
  const hipStream_t stream = (hipStream_t)hip_stream;
  const hipError_t e = dtype == TFGFA_DTYPE_BF16 ? launch_shared<__bf16>(a, x, B * H, stream)
                                                 : launch_shared<_Float16>(a, x, B * H, stream);
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
