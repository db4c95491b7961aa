// tfgfa_paged.hip - one decode step of attention over a paged key-value cache, MI355X (gfx950), bf16 or fp16, head
// dims that are multiples of 8 up to 128, query heads sharing key-value heads.
//
// For each query head h of key-value head h' (G = H / H_kv of them):
//     x_j = scale q_h . k_j,   o_h = sum_j e^(x_j) v_j / sum_j e^(x_j),   lse_h = log sum_j e^(x_j)
// over the rows j < L of the sequence, row j being row j % page of page table[j / page].
//
// Bound: HBM.  Each K and V row is read once, 4D bytes for 4DG flops.  The 16 columns of a 16x16 matrix tile are the
// query heads of one key-value head, so that up to 16 of them cost what one does:
//   scores   S^T[key][head] = K Q^T      v_mfma_f32_16x16x32 (products exact, float32 sums)
//   output   O^T[dim][head] += V^T P^T   the same, P as a sum of three bf16 or two fp16
// A wave takes 32 keys at a time.  The scores leave the first product with lane (g = lane / 16, i = lane % 16)
// holding keys 4g .. 4g + 3 of each 16 for head i; two such sets are the second product's B operand as they stand
// (the contraction runs over keys, whose order is free).  Its A operand wants 8 keys' values of one dim in a lane:
// the lane loads kDV neighbouring dims of each of the 8 rows, and byte permutes put the keys of a dim side by side.
// So neither P nor V moves between lanes.  P is split into parts of the element type, each what rounding left of the
// ones before: three of bf16 hold all 24 bits of a float32, two of fp16 miss 2^-23 of it at most, twice a float32's
// rounding.  (fp16 ends at 2^-24: its P goes in times 2^13, so that weights are kept to 2^-38 of the largest.)  An
// infinite V makes NaN of a part of 0 or below; a wave whose sums hold NaN takes its keys again with the first part
// alone, for those sums.  (With P and V as float32 on v_mfma_f32_16x16x4_f32 a block of 32 keys took 1024 matrix
// cycles at D = 64 instead of 192 with two parts.  Two of bf16, 16 bits, gave one output in a thousand another
// rounding than the definition's; the third takes 32 sequences of 25 heads of 1024 rows from 28.7 to 29.3 us, one of
// 12 heads of 400 from 6.45 to 6.65, and caches that are divided nothing.)
//
// Division of the work.  A unit is a (sequence, key-value head, 16 query heads).  The lengths are known on the device
// only, so every workgroup works the division out from them (plan, below): one chunk length C for all units, with
// about `target` workgroups in all; a unit of more than C rows is divided over several workgroups.  Each leaves its
// part (sums of weighted values and of weights, and their offset) in the workspace, and the one that arrives last
// joins them (arrival words and memory order as in tfgfa_decode.hip) and, where it is asked for, adds the unit's key
// weights from the scores that the parts have left: e^(scale (s - m)) / W, s without the scale, m the offset of the
// joined sums and W their sum of weights, so that s - m is exact for near scores of any size (with e^(x - lse) of
// rounded x and lse, weights of scores near 2^23 were off by tens of percent).
//
// Measured, inputs that no cache holds: 32 sequences of 25 heads, D = 64, lengths to 1024, 120 MB in 28.6 us (24.5
// from the Infinity Cache; a plain read of as many bytes 21.6); 4 sequences of 32 heads on 8, D = 128, to 32768 rows,
// 385 MB in 80 us (67); one sequence of 12 heads, 400 rows, 6.5 us (the chain length - pages - K - V - output; 1.6 us
// are the launch); 4 sequences of 16 heads to 4096 rows with key weights, 50 MB, 23 us, 4 of them the weights (10).
// Matrix units busy 7%, VALU issue 19%, 76% of the wave cycles in waits at the first: loads under way bound it, and
// their number is what the registers hold (a second set of them 192 to 256 VGPRs, slower; 4 waves a SIMD spill; blocks
// of 64 keys, 8 or 16 waves a workgroup, slower).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tfgfa.h"
#include "tfgfa_arrive.h"
#include "tfgfa_layout.h"
#include "tfgfa_serving.h"

namespace tfgfa_paged {

using tfgfa::apart;
using tfgfa::Pages;
using tfgfa::pages_apart;
using tfgfa::pages_ok;
using tfgfa::Vecs;
using tfgfa::vecs_ok;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned long long u64;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxD = 128;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kHeads = 16;                    // query heads of a unit
constexpr int kTile = 16;                     // keys of a matrix tile
constexpr int kTiles = 2;                     // tiles of a wave's block (one contraction of P V)
constexpr int kBlock = kTile * kTiles;        // keys of a wave's block
constexpr int kGranule = kWaves * kBlock;     // keys of a workgroup's block
constexpr int kMaxParts = 64;                 // workgroups of a unit
// A buffer offset past any num_records built here: the load returns zero without a memory access.
constexpr uint32_t kOutOfRange = 0x7FFFFFF0u;
constexpr int kScoreTail = 4;                 // a head's scores end with a place for the new row's
constexpr int kPolicyCoherent = 16;           // buffer loads from the device's coherence point (sc1)

template <class T>
struct Elem;
// kParts: of the type that a P is split into; kShift: it goes in times 2^kShift.  kSlack: how far a score may pass its
// head's offset; e^kSlack 2^kShift is a number of the type.
template <>
struct Elem<__bf16> {
  static constexpr int kParts = 3, kShift = 0;
  static constexpr float kSlack = 8.f;
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                   c, 0, 0, 0);
  }
};
template <>
struct Elem<_Float16> {
  static constexpr int kParts = 2, kShift = 13;
  static constexpr float kSlack = 2.f;
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                  0, 0, 0);
  }
};

// Two values of the element type in 32 bits; *rest: what rounding left of them.  (bf16 by cutting off, which is two
// operations less in a row and leaves no part below 0.)
template <class T>
__device__ __forceinline__ uint32_t pack(float x, float y, float* rx, float* ry) {
  if constexpr (std::is_same_v<T, __bf16>) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    *rx = x - __uint_as_float(a & 0xFFFF0000u);
    *ry = y - __uint_as_float(b & 0xFFFF0000u);
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
  }
  const typename Elem<T>::x2 z = {(T)x, (T)y};
  *rx = x - (float)z[0];
  *ry = y - (float)z[1];
  return __builtin_bit_cast(uint32_t, z);
}
// (x.lo16, y.lo16) and (x.hi16, y.hi16): one dim of two keys side by side (v_perm_b32).
__device__ __forceinline__ uint32_t pair_lo(uint32_t x, uint32_t y) {
  return __builtin_amdgcn_perm(y, x, 0x05040100u);
}
__device__ __forceinline__ uint32_t pair_hi(uint32_t x, uint32_t y) {
  return __builtin_amdgcn_perm(y, x, 0x07060302u);
}

// e^x as 2^(x log2 e), the difference of two scores taken first: scores up to the largest float keep their place.
// v_exp_f32: results below 2^-126 are 0.
__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ float log_(float x) { return log2f(x) * kLn2; }
// 1 / x to a rounding for the normal x > 0 whose inverse is normal: v_rcp_f32 is off by one unit, a Newton step takes
// it away.  (The compiler's division is 10 instructions one after another.)
__device__ __forceinline__ float inverse(float x) {
  const float y = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, y, 1.f), y, y);
}

// What turns a head's scores into its key weights: their offset, and one over the sum of e^(scale (s - offset)); 0 for
// a head whose log-sum-exp is not finite, which adds nothing.
struct alignas(8) Share {
  float offset, inverse;
};
// w and the key weight of score s.
__device__ __forceinline__ float add_weight(float w, float s, Share head, float scale_log2) {
  const float p = __builtin_amdgcn_exp2f((s - head.offset) * scale_log2);
  return head.inverse != 0.f ? fmaf(p, head.inverse, w) : w;
}

// Floats of a part.
__host__ __device__ constexpr long long part_floats(int D) { return (long long)kHeads * (D + 2); }

struct Args {
  const char* k;
  const char* v;
  const void* kn;
  const void* vn;
  void* o;
  float* lse;       // natural log, or null
  char* arrive;
  float* part;      // per workgroup of a divided unit: [head][D] sums, then [head] their offsets, [head] of weights
  Share* shares;    // (B, H) for the weights, or null
  float* scores;    // (B, H, n_pad) scores without the scale, the new row's at n_pad - kScoreTail, or null
  u64 tag;
  Pages ks, vs;
  Vecs qs, os, kns, vns;
  long long n_pad;
  float scale, scale_log2;
  float slack;      // Elem::kSlack in scores without the scale
  int H, G, P, page, D;
  int tiles;        // 16-head tiles of a key-value head
  int min_granules; // smallest part
  float* weights;   // key_weights where the workgroup that ends a unit adds them, or null; strides
  long long wb, wh;
};

// The arguments that a kernel has before Args.  units: of one sequence, Hkv * tiles; target: parts of a unit that the
// division aims at over all sequences (0: none are divided); j / page = j * div_m >> div_s for j < 2^31.
struct First {
  const int* table;
  const int* lens;
  long long table_stride;
  const void* q;
  int n_max;
  uint32_t div_m;
  int div_s, target, units, B;
};

// Sum of x over the lanes up to and with this one (row shifts inside 16 lanes, then the rows' ends).
template <int kCtrl, int kRows>
__device__ __forceinline__ int add_dpp(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, kCtrl, kRows, 0xF, false);
}
__device__ __forceinline__ int scan64(int x) {
  x = add_dpp<0x111, 0xF>(x);
  x = add_dpp<0x112, 0xF>(x);
  x = add_dpp<0x114, 0xF>(x);
  x = add_dpp<0x118, 0xF>(x);
  x = add_dpp<0x142, 0xA>(x);  // lane 15 of rows 0 and 2 to the row after
  return add_dpp<0x143, 0xC>(x);  // lane 31 to rows 2 and 3
}

struct Piece {
  int b, unit, s, S;  // sequence, unit of it, part s of S
  int first;          // the unit's first workgroup
  int len;            // cache_seqlens[b]
};

__device__ __forceinline__ int granules(int rows) { return (rows + kGranule - 1) / kGranule; }

// x / y for 0 <= x < 2^21, y > 0: the product's error, 2^-22 of it, is below the 0.5 / y that x + 0.5 is away from the
// next quotient.  (The compiler's exact division is some 40 instructions, a microsecond for a few of them in a row.)
__device__ __forceinline__ int quot(int x, int y) {
  return (int)(((float)x + 0.5f) * __builtin_amdgcn_rcpf((float)y));
}

// The piece of work of workgroup w of a batch whose sequences are divided: with C = ceil(all granules / target)
// granules to a part, sequence b takes ceil(granules_b / C) workgroups (one at least, to write the empty row) for each
// of its units, in the order of (sequence, unit, part).  Every wave works it out alike; false where no work is left.
__device__ __forceinline__ bool plan(const int* lens, int B, int most, int append, int units, int target,
                                     int min_granules, int w, int lane, Piece* out) {
  // Granules of a sequence of n cached rows, of which more than `most` do not fit.
  auto of = [&](int n) { return n >= 0 && n <= most ? granules(n + append) : 0; };
  int total = 0;
  int n0 = 0, g0 = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int n = b0 + lane < B ? lens[b0 + lane] : 0;
    const int g = of(n);
    total += __builtin_amdgcn_readlane(scan64(g), 63);
    if (b0 == 0) n0 = n, g0 = g;
  }
  const int C = max(min_granules, quot(total + target - 1, target));
  int before = 0;  // parts of one unit in the sequences before
  for (int b0 = 0; b0 < B; b0 += 64) {
    int n = n0, g = g0;
    if (b0 > 0) {
      n = b0 + lane < B ? lens[b0 + lane] : 0;
      g = of(n);
    }
    const int S = b0 + lane < B ? max(1, min(kMaxParts, quot(g + C - 1, C))) : 0;
    const int upto = before + scan64(S);
    const u64 done = __builtin_amdgcn_ballot_w64(upto * units <= w);
    const int at = __builtin_popcountll(done);
    if (at < 64 && b0 + at < B) {
      const int Sb = __builtin_amdgcn_readlane(S, at);
      const int first = (__builtin_amdgcn_readlane(upto, at) - Sb) * units;
      const int i = w - first;
      out->b = b0 + at;
      out->unit = quot(i, Sb);
      out->s = i - out->unit * Sb;
      out->S = Sb;
      out->first = first + out->unit * Sb;
      out->len = __builtin_amdgcn_readlane(n, at);
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, int nbytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, nbytes, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
template <int kN>
__device__ __forceinline__ void load_v(uint32_t (&x)[kN], __amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (kN == 4) {
    const u32x4 y = load16(r, off);
    x[0] = y[0], x[1] = y[1], x[2] = y[2], x[3] = y[3];
  } else {
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
    x[0] = y[0], x[1] = y[1];
  }
}
template <int kN>
__device__ __forceinline__ void load_v(uint32_t (&x)[kN], const char* p) {
  if constexpr (kN == 4) {
    const u32x4 y = *reinterpret_cast<const u32x4*>(p);
    x[0] = y[0], x[1] = y[1], x[2] = y[2], x[3] = y[3];
  } else {
    const u32x2 y = *reinterpret_cast<const u32x2*>(p);
    x[0] = y[0], x[1] = y[1];
  }
}

// The sum (and the largest) of x over the four lanes of a head, in all of them: lanes 16 and 32 apart, by exchanges of
// 16-lane rows between two registers.
template <class F>
__device__ __forceinline__ float over_rows(float x, F f) {
  const uint32_t a = __float_as_uint(x);
  const auto y = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t b = __float_as_uint(f(__uint_as_float(y[0]), __uint_as_float(y[1])));
  const auto z = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return f(__uint_as_float(z[0]), __uint_as_float(z[1]));
}

// The same over the 64 lanes: rotations inside 16 lanes, then their rows.
template <class F>
__device__ __forceinline__ float over_lanes(float x, F f) {
  auto turn = [&](auto c) {
    x = f(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(c)::value, 0xF, 0xF, false)));
  };
  turn(std::integral_constant<int, 0x121>());
  turn(std::integral_constant<int, 0x122>());
  turn(std::integral_constant<int, 0x124>());
  turn(std::integral_constant<int, 0x128>());
  return over_rows(x, f);
}

// The tables and lengths are not written while a step runs: those at uniform places come by scalar loads.
typedef const __attribute__((address_space(4))) int* uniform_ints;

// kDV: dims of a lane in V, 4 (D <= 64) or 8.  kFull: D == 16 kDV.  kSpan: keys that are sure to be in one page: a
// tile (16) where the page size is a multiple of it, otherwise 1, whose lanes have an address each (5 to 20% slower
// on pages that allow both).  kFused: this kernel adds key weights.  kDivide: sequences may be divided (grid: flat;
// otherwise units by sequences). The first 14 dwords of the arguments are preloaded into scalar registers
// (-amdgpu-kernarg-preload-count): what the first loads, of the length and of the first block's pages, wait for.
template <class T, int kDV, bool kFull, int kSpan, bool kDivide, bool kFused>
__global__ __launch_bounds__(kThreads, 2) void paged_kernel(const int* __restrict__ table, const int* __restrict__ lens,
                                                            long long table_stride, const T* __restrict__ q, int n_max,
                                                            uint32_t div_m, int div_s, int target, int units, int B,
                                                            const Args a) {
  constexpr int kDP = kDV / 2;          // pieces of 32 dims
  constexpr int kDm = 16 * kDV;
  constexpr int kRow = kDm + 4;
  // The waves' outputs; later the shares of a unit's parts and the sums of the groups that join them.
  constexpr int kLds = kWaves * kHeads * kRow, kLdsJoin = kHeads * kMaxParts + 4 * kThreads;
  __shared__ __attribute__((aligned(16))) float sh_o[kLds > kLdsJoin ? kLds : kLdsJoin];
  __shared__ float sh_m[kWaves][kHeads], sh_l[kWaves][kHeads];
  __shared__ Share sh_share[kHeads];
  __shared__ int sh_last;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, i = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int append = a.kn != nullptr;
  auto page_of = [&](int j) { return (int)(((u64)(uint32_t)j * div_m) >> div_s); };
  Piece pc;
  if (!kDivide) {
    pc.b = blockIdx.y, pc.unit = blockIdx.x;
    pc.s = 0, pc.S = 1;
  } else if (B == 1) {  // part s takes granules s, s + S, ..: where it starts does not depend on the length
    pc.b = 0;
    pc.unit = quot(blockIdx.x, target);
    pc.first = pc.unit * target;
    pc.s = blockIdx.x - pc.first;
  } else if (!plan(lens, B, n_max - append, append, units, target, a.min_granules, blockIdx.x, lane, &pc)) {
    return;
  }
  const int b = __builtin_amdgcn_readfirstlane(pc.b), unit = __builtin_amdgcn_readfirstlane(pc.unit);
  const int s_mine = __builtin_amdgcn_readfirstlane(pc.s);

  // The first block's pages are looked up beside the length: where it starts does not depend on it.
  const int kb0 = (s_mine * kWaves + wave) * kBlock;
  const int* const row = table + (long long)b * table_stride;
  constexpr int kIds = kSpan == 1 ? 1 : kBlock / kSpan;
  auto look_up = [&](int (&id)[kIds], int at) {
    if constexpr (kSpan > 1) {
#pragma unroll
      for (int c = 0; c < kIds; ++c)
        id[c] = __builtin_amdgcn_readfirstlane(at + c * kSpan < n_max ? ((uniform_ints)row)[page_of(at + c * kSpan)] : -1);
    } else {  // lane l: key at + l % kBlock
      const int key = at + (lane & (kBlock - 1));
      id[0] = key < n_max ? row[page_of(key)] : -1;
    }
  };
  int ids[kIds];
  look_up(ids, kb0);
  const int len = kDivide && B > 1 ? __builtin_amdgcn_readfirstlane(pc.len) : ((uniform_ints)lens)[b];

  // The other arguments, needed next: their loads go out with the ones above rather than where they are used.
  asm volatile("" ::"s"(a.k), "s"(a.v), "s"(a.ks.p), "s"(a.ks.h), "s"(a.ks.n), "s"(a.vs.p), "s"(a.vs.h), "s"(a.vs.n),
               "s"(a.qs.b), "s"(a.qs.h));

  // Queries: the B operand, head i, zero past the unit's heads and past D.
  const int D = a.D;
  const int kv = a.tiles == 1 ? unit : __builtin_amdgcn_readfirstlane(quot(unit, a.tiles)), tile = unit - kv * a.tiles;
  const int h0 = kv * a.G + tile * kHeads;               // first query head
  const int nh = min(kHeads, a.G - tile * kHeads);       // query heads of the unit
  u32x4 qf[kDP];
  {
    const __amdgpu_buffer_rsrc_t qr = rows_rsrc(q + b * a.qs.b + h0 * a.qs.h, INT32_MAX / 2);
#pragma unroll
    for (int p = 0; p < kDP; ++p)
      qf[p] = load16(qr, i < nh && (kFull || 32 * p + 8 * g < D) ? (uint32_t)(i * (int)a.qs.h * 2 + 64 * p + 16 * g)
                                                                 : kOutOfRange);
  }
  u64* const aw = reinterpret_cast<u64*>(a.arrive + ((long long)b * units + unit) * tfgfa::kArriveStride);
  const bool valid = len >= 0 && len <= n_max - append;
  const int Lr = valid ? len : 0;                        // rows that are in the cache
  const int L = valid ? len + append : 0;                // rows attended to
  const int S = !kDivide   ? 1
                : B == 1 ? max(1, min(target, quot(granules(L) + a.min_granules - 1, a.min_granules)))
                         : __builtin_amdgcn_readfirstlane(pc.S);
  if (kDivide && s_mine >= S) return;
  u64 aw_start = 0;
  if (kDivide && S > 1 && wave == 0) aw_start = __hip_atomic_load(aw, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // The blocks of this wave: those of its part's cached rows, and in the unit's last wave one more for the new row,
  // which is read from the arguments (no wave reads its place in the cache, which this one writes).
  const int stride = S * kGranule;
  const int after = kb0 < Lr ? granules(Lr - kb0) : 0;
  const int blocks = S == 1 ? after : quot(after + S - 1, S);
  const int all = blocks + (append && valid && s_mine == S - 1 && wave == kWaves - 1 ? 1 : 0);
  struct Block {
    int at, rows;  // first key and how many of the block's keys there are
    bool fresh;    // the new row
  };
  auto block = [&](int n) {
    const int at = kb0 + n * stride;
    return n < blocks ? Block{at, min(kBlock, Lr - at), false} : Block{Lr, 1, true};
  };

  const char* const kh = a.k + kv * a.ks.h;
  const char* const vh = a.v + kv * a.vs.h;
  const char* const kn = append ? reinterpret_cast<const char*>(static_cast<const T*>(a.kn) + b * a.kns.b + kv * a.kns.h) : kh;
  const char* const vn = append ? reinterpret_cast<const char*>(static_cast<const T*>(a.vn) + b * a.vns.b + kv * a.vns.h) : vh;
  // Loads of a block.  Rows that are not there come as zeros (kSpan > 1: past the buffer, which for the new row ends
  // before a second one; otherwise the loads go to a row that is there, and V is cleared below); so do dims past D
  // in K.
  u32x4 k[kTiles][kDP];           // row i of a tile, dims 32p + 8g .. of piece p: the A operand of the scores
  uint32_t v[kTiles][4][kDP];     // row 4g + r of a tile, dims kDV i ..
  const uint32_t k_lane = (uint32_t)(i * (int)a.ks.n + 16 * g);
  const uint32_t v_lane = (uint32_t)(4 * g * (int)a.vs.n + 2 * kDV * i);
  // Rows [at, at + kSpan) of the block in page id, as a buffer of those that there are.
  auto span = [&](const Block& x, int c, int id, const char* base, const char* fresh, const Pages& st) {
    const bool in = (uint32_t)id < (uint32_t)a.P;
    const int key = x.at + c * kSpan, rows = max(0, min(kSpan, x.rows - c * kSpan));
    const u64 pid = (uint32_t)(in ? id : 0), off = (uint32_t)(key - page_of(key) * a.page);
    const u64 where = (u64)(uintptr_t)base + pid * (u64)st.p + off * (uint32_t)st.n;
    const u64 start = x.fresh ? (u64)(uintptr_t)fresh : where;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)start);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(start >> 32));
    return rows_rsrc(reinterpret_cast<const char*>((u64)hi << 32 | lo),
                     __builtin_amdgcn_readfirstlane(in || x.fresh ? rows * (int)st.n : 0));
  };
  // The row of key l % kBlock of the block.
  auto one = [&](const Block& x, int id, const char* base, const char* fresh, const Pages& st) {
    const int key = lane & (kBlock - 1);
    const bool in = (uint32_t)id < (uint32_t)a.P && key < x.rows;
    const u64 pid = in ? id : 0, off = in ? x.at + key - page_of(x.at + key) * a.page : 0;
    return x.fresh ? (u64)(uintptr_t)fresh : (u64)(uintptr_t)base + pid * (u64)st.p + off * (uint32_t)st.n;
  };
  auto load_keys = [&](const Block& x, const int (&id)[kIds]) {
    if constexpr (kSpan > 1) {
#pragma unroll
      for (int c = 0; c < kIds; ++c) {
        const __amdgpu_buffer_rsrc_t kr = span(x, c, id[c], kh, kn, a.ks);
#pragma unroll
        for (int t = c * kSpan / kTile; t < (c + 1) * kSpan / kTile; ++t)
#pragma unroll
          for (int p = 0; p < kDP; ++p)
            k[t][p] = load16(kr, kFull || 32 * p + 8 * g < D
                                     ? k_lane + (t - c * kSpan / kTile) * kTile * (uint32_t)a.ks.n + 64 * p
                                     : kOutOfRange);
      }
    } else {
      const u64 at = one(x, id[0], kh, kn, a.ks);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const char* const kr = reinterpret_cast<const char*>(__shfl(at, t * kTile + i));
#pragma unroll
        for (int p = 0; p < kDP; ++p)
          k[t][p] = *reinterpret_cast<const u32x4*>(kr + (kFull || 32 * p + 8 * g < D ? 64 * p + 16 * g : 0));
      }
    }
  };
  auto load_values = [&](const Block& x, const int (&id)[kIds]) {
    if constexpr (kSpan > 1) {
#pragma unroll
      for (int c = 0; c < kIds; ++c) {
        const __amdgpu_buffer_rsrc_t vr = span(x, c, id[c], vh, vn, a.vs);
#pragma unroll
        for (int t = c * kSpan / kTile; t < (c + 1) * kSpan / kTile; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            load_v(v[t][r], vr, kFull || kDV * i < D
                                    ? v_lane + ((t - c * kSpan / kTile) * kTile + r) * (uint32_t)a.vs.n
                                    : kOutOfRange);
      }
    } else {
      const u64 at = one(x, id[0], vh, vn, a.vs);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          load_v(v[t][r], reinterpret_cast<const char*>(__shfl(at, t * kTile + 4 * g + r)) +
                              (kFull || kDV * i < D ? 2 * kDV * i : 0));
    }
  };

  float m, l;
  f32x4 acc[kDV];
  // All parts of P: 1 or 0, kept in a scalar register.  (A branch on what the compiler takes for a value of each lane
  // only masks lanes, and a matrix instruction runs whatever the mask.)
  int every = __builtin_amdgcn_readfirstlane(1);
  // The wave's sums into LDS.  acc[j], register r of lane (g, i): dim kDV (4g + r) + j of head i.
  auto leave = [&]() {
    if (i < nh) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < kDV; j += 4)
          *reinterpret_cast<f32x4*>(&sh_o[(wave * kHeads + i) * kRow + kDV * (4 * g + r) + j]) =
              f32x4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
    }
  };

  // The arithmetic of block x.  kMore: another block follows, whose K goes out once the scores have read this one's,
  // and its V once the output has, so that one of the two is always in flight with one set of registers.
  auto step = [&](const Block& x, const Block& y, auto more) {
      constexpr bool kMore = decltype(more)::value;
      int next[kIds];
      if constexpr (kMore) look_up(next, y.at);
      if (!kFull && kSpan == 1)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int p = 0; p < kDP; ++p)
            if (32 * p + 8 * g >= D) k[t][p] = u32x4{0, 0, 0, 0};
      // The new row goes to its page from the lanes of the block's first key; without a page its score is NaN.
      const int home = x.fresh && tile == 0 ? __builtin_amdgcn_readfirstlane(ids[0]) : -1;
      const bool write = (uint32_t)home < (uint32_t)a.P;
      const u64 row_in = write ? Lr - page_of(Lr) * a.page : 0;
      if (write && i == 0) {
        char* const to = const_cast<char*>(kh) + (u64)home * (u64)a.ks.p + row_in * (uint32_t)a.ks.n + 16 * g;
#pragma unroll
        for (int p = 0; p < kDP; ++p)
          if (kFull || 32 * p + 8 * g < D) *reinterpret_cast<u32x4*>(to + 64 * p) = k[0][p];
      }
      float s[kTiles][4];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < kDP; ++p) c = Elem<T>::mfma(k[t][p], qf[p], c);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = c[r];
      }
      if constexpr (kMore) load_keys(y, next);
      __builtin_amdgcn_sched_barrier(0);
      // (Scores without the scale.)  NaN through a page outside the pool (a bit each of the block's spans), -inf where
      // there is no key.
      u64 out = 0;
      if constexpr (kSpan > 1) {
#pragma unroll
        for (int c = 0; c < kIds; ++c) out |= (u64)((uint32_t)ids[c] >= (uint32_t)a.P) << c;
      } else {
        out = __builtin_amdgcn_ballot_w64((uint32_t)ids[0] >= (uint32_t)a.P);
      }
      if (x.rows < kBlock || out) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = t * kTile + 4 * g + r;
            if ((out >> (kSpan > 1 ? t * kTile / kSpan : key)) & 1u) s[t][r] = __uint_as_float(0x7FC00000u);
            if (key >= x.rows) s[t][r] = -INFINITY;
          }
      }
      if (a.scores != nullptr && i < nh) {
        if constexpr (kFused) {  // for the workgroup that ends the unit, to the coherence point
          const __amdgpu_buffer_rsrc_t sr = rows_rsrc(a.scores + ((long long)b * a.H + h0) * a.n_pad, INT32_MAX / 2);
          const int head = i * (int)a.n_pad;
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const f32x4 y = {s[t][0], s[t][1], s[t][2], s[t][3]};
            const int at = x.fresh ? (t == 0 && g == 0 ? head + (int)a.n_pad - kScoreTail : -1)
                                   : (t * kTile < x.rows ? head + x.at + t * kTile + 4 * g : -1);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), sr,
                                                   at < 0 ? (int)kOutOfRange : at * 4, 0, kPolicyCoherent);
          }
        } else {
          float* const to = a.scores + ((long long)b * a.H + h0 + i) * a.n_pad;
          if (x.fresh) {
            if (g == 0) to[a.n_pad - kScoreTail] = s[0][0];
          } else {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              if (t * kTile < x.rows)
                *reinterpret_cast<f32x4*>(to + x.at + t * kTile + 4 * g) =
                    f32x4{s[t][0], s[t][1], s[t][2], s[t][3]};
          }
        }
      }
      // The offset of each head moves only when a score passes it by the slack, so that lanes compare notes in few
      // blocks.  (By the difference, which is exact for near scores: m + slack may round up by more than fp16 has room.)
      float mb = s[0][0];
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) mb = fmaxf(mb, s[t][r]);
      if (__builtin_amdgcn_ballot_w64(mb - m > a.slack)) {
        mb = over_rows(mb, [](float u, float w) { return fmaxf(u, w); });
        const float mn = fmaxf(m, mb);
        const float f = m == -INFINITY ? 0.f : exp_((m - mn) * a.scale);
        l *= f;
#pragma unroll
        for (int j = 0; j < kDV; ++j) acc[j] *= f;
        m = mn;
      }
      const float mu = m == -INFINITY ? 0.f : m;
      constexpr int kParts = Elem<T>::kParts;
      u32x4 part[kParts][kTiles / 2];
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          float p0 = __builtin_amdgcn_exp2f((s[t][r] - mu) * a.scale_log2);
          float p1 = __builtin_amdgcn_exp2f((s[t][r + 1] - mu) * a.scale_log2);
          l += p0 + p1;
          p0 *= 1 << Elem<T>::kShift, p1 *= 1 << Elem<T>::kShift;
#pragma unroll
          for (int c = 0; c < kParts; ++c) part[c][t / 2][2 * (t % 2) + r / 2] = pack<T>(p0, p1, &p0, &p1);
        }
      if (write && g == 0 && (kFull || kDV * i < D)) {
        char* const to = const_cast<char*>(vh) + (u64)home * (u64)a.vs.p + row_in * (uint32_t)a.vs.n + 2 * kDV * i;
        if constexpr (kDV == 8)
          *reinterpret_cast<u32x4*>(to) = u32x4{v[0][0][0], v[0][0][1], v[0][0][2], v[0][0][3]};
        else
          *reinterpret_cast<u32x2*>(to) = u32x2{v[0][0][0], v[0][0][1]};
      }
      if (kSpan == 1 && x.rows < kBlock)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t * kTile + 4 * g + r >= x.rows)
#pragma unroll
              for (int e = 0; e < kDP; ++e) v[t][r][e] = 0;
#pragma unroll
      for (int t = 0; t < kTiles; t += 2)
#pragma unroll
        for (int e = 0; e < kDP; ++e) {
          const auto& va = v[t];
          const auto& vb = v[t + 1];
          const u32x4 v0 = {pair_lo(va[0][e], va[1][e]), pair_lo(va[2][e], va[3][e]), pair_lo(vb[0][e], vb[1][e]),
                            pair_lo(vb[2][e], vb[3][e])};
          const u32x4 v1 = {pair_hi(va[0][e], va[1][e]), pair_hi(va[2][e], va[3][e]), pair_hi(vb[0][e], vb[1][e]),
                            pair_hi(vb[2][e], vb[3][e])};
          acc[2 * e] = Elem<T>::mfma(v0, part[0][t / 2], acc[2 * e]);
          acc[2 * e + 1] = Elem<T>::mfma(v1, part[0][t / 2], acc[2 * e + 1]);
          if (__builtin_amdgcn_readfirstlane(every)) {
#pragma unroll
            for (int c = 1; c < kParts; ++c) {
              acc[2 * e] = Elem<T>::mfma(v0, part[c][t / 2], acc[2 * e]);
              acc[2 * e + 1] = Elem<T>::mfma(v1, part[c][t / 2], acc[2 * e + 1]);
            }
          }
        }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kMore) {
        load_values(y, next);
#pragma unroll
        for (int c = 0; c < kIds; ++c) ids[c] = next[c];
      }
  };
  for (;;) {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < kDV; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (all == 0) break;
    Block x = block(0);
    if (x.fresh) look_up(ids, Lr);
    load_keys(x, ids);
    load_values(x, ids);
#pragma unroll 1
    for (int n = 1; n < all; ++n) {
      const Block y = block(n);
      step(x, y, std::true_type());
      x = y;
    }
    step(x, x, std::false_type());
    float any = 0.f;  // NaN if one of the sums is
#pragma unroll
    for (int j = 0; j < kDV; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) any = fmaf(acc[j][r], 0.f, any);
    if (!__builtin_amdgcn_readfirstlane(every) || !__builtin_amdgcn_ballot_w64(any != any)) break;
    leave();  // (the sums that are not NaN are kept)
    every = __builtin_amdgcn_readfirstlane(0);
    look_up(ids, kb0);
  }
  if (kDivide && S > 1 && wave == 0 && lane == 0 && (aw_start >> tfgfa::kTagShift) != a.tag) {
    u64 expected = aw_start;
    __hip_atomic_compare_exchange_strong(aw, &expected, a.tag << tfgfa::kTagShift, __ATOMIC_RELAXED,
                                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }

  // key_weights of the unit's heads (no other unit has this key-value head), by the workgroup that ends it and has left
  // their shares in LDS.
  auto add_weights = [&]() {
    const __amdgpu_buffer_rsrc_t wr = rows_rsrc(a.weights + b * a.wb + kv * a.wh, INT32_MAX / 2);
    const __amdgpu_buffer_rsrc_t sr = rows_rsrc(a.scores + ((long long)b * a.H + h0) * a.n_pad, INT32_MAX / 2);
    auto store = [&](float x, int at) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), wr, at < 0 ? (int)kOutOfRange : at * 4, 0, 0);
    };
    if (append && wave == kWaves - 1) {  // the new row's
      const Share head = lane < nh ? sh_share[lane] : Share{0.f, 0.f};
      const float x = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
          sr, lane < nh ? (lane * (int)a.n_pad + (int)a.n_pad - kScoreTail) * 4 : (int)kOutOfRange, 0, kPolicyCoherent));
      const float w = over_lanes(add_weight(0.f, x, head, a.scale_log2), [](float u, float v) { return u + v; });
      store(w, lane == 0 && (uint32_t)((uniform_ints)row)[page_of(Lr)] < (uint32_t)a.P ? Lr : -1);
    }
    // Four rows a thread; kItems heads of such blocks of rows in flight at once.
    constexpr int kItems = 8;
    const int items = (Lr + 4 * kThreads - 1) / (4 * kThreads) * nh;
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    int h = 0, j = 4 * tid;
    for (int n = 0; n < items; n += kItems) {
      u32x4 x[kItems], y[kItems];
      int hx = h, jx = j;
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        x[u] = __builtin_amdgcn_raw_buffer_load_b128(sr, jx < Lr ? (hx * (int)a.n_pad + jx) * 4 : (int)kOutOfRange, 0,
                                                     kPolicyCoherent);
        y[u] = load16(wr, jx < Lr && hx == nh - 1 ? jx * 4 : kOutOfRange);
        if (++hx == nh) hx = 0, jx += 4 * kThreads;
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const Share head = sh_share[h];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = add_weight(w[e], __uint_as_float(x[u][e]), head, a.scale_log2);
        if (++h == nh) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            store(__uint_as_float(y[u][e]) + w[e], j + e < Lr ? j + e : -1);
            w[e] = 0.f;
          }
          h = 0, j += 4 * kThreads;
        }
      }
    }
  };

  // Join the waves.  (Offsets without the scale: differences first, here too.)
  l = over_rows(l, [](float u, float w) { return u + w; });
  if (!every && i < nh) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < kDV; ++j) {
        const float first = sh_o[(wave * kHeads + i) * kRow + kDV * (4 * g + r) + j];
        if (first == first) acc[j][r] = first;
      }
  }
  leave();
  if (i < nh && g == 0) {
    sh_m[wave][i] = m;
    sh_l[wave][i] = l;
  }
  __syncthreads();
  const long long part = part_floats(D);
  float* const mine = a.part + blockIdx.x * part;
  const float nan = __uint_as_float(0x7FC00000u);
  for (int e = tid; e < nh * kDm; e += kThreads) {
    const int h = e / kDm, d = e % kDm;
    if (!kFull && d >= D) continue;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sh_m[w][h]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float lt = 0.f, ot = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp_((sh_m[w][h] - Mu) * a.scale);
      lt = fmaf(f, sh_l[w][h], lt);
      ot = fmaf(f, sh_o[(w * kHeads + h) * kRow + d], ot);
    }
    ot *= 1.f / (1 << Elem<T>::kShift);
    if (S > 1) {
      __hip_atomic_store(mine + h * D + d, ot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d < 2)
        __hip_atomic_store(mine + (D + d) * kHeads + h, d == 0 ? M : lt, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else {
      const float on = lt == 0.f ? 0.f : ot * inverse(lt);
      static_cast<T*>(a.o)[b * a.os.b + (h0 + h) * a.os.h + d] = (T)(valid ? on : nan);
      if (d == 0 && (a.lse || a.shares || kFused)) {
        const float ls = lt == 0.f ? -INFINITY : fmaf(Mu, a.scale, log_(lt));
        const Share head = {Mu, fabsf(ls) < INFINITY ? inverse(lt) : 0.f};
        if (a.lse) a.lse[(long long)b * a.H + h0 + h] = valid ? ls : nan;
        if (a.shares) a.shares[(long long)b * a.H + h0 + h] = head;
        if (kFused) sh_share[h] = head;
      }
    }
  }
  if (!kDivide || S == 1) {
    if (kFused && valid) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's scores
      __syncthreads();
      add_weights();
    }
    return;
  }
  // The part is at the coherence point once its stores are acknowledged; then the arrival is counted.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const u64 old = __hip_atomic_fetch_add(aw, (u64)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int last = (old & ((1ull << tfgfa::kTagShift) - 1)) == (u64)(S - 1);
    if (last) __hip_atomic_store(aw, (u64)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh_last = last;
  }
  __syncthreads();
  if (!sh_last) return;
  asm volatile("" ::: "memory");
  // Join the parts (sums with offset m): their shares e^(m_s - M) / sum into LDS, a wave a head; then 4 dims a thread,
  // the parts dealt to groups of threads whose sums are added in order.  The first parts' loads go out before the
  // shares are known.
  const __amdgpu_buffer_rsrc_t parts = rows_rsrc(a.part + pc.first * part, (int)(S * part * 4));
  auto coherent = [&](int at) {
    return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(parts, at, 0, kPolicyCoherent));
  };
  constexpr int kQuads = kDm / 4, kBatch = 8;
  const int quads = nh * kQuads;
  const int join = max(1, kThreads / quads);  // groups
  const int grp = join > 1 ? tid / quads : 0;
  auto fetch = [&](u32x4 (&z)[kBatch], int e, int s0) {
    const int h = e / kQuads, d = e % kQuads * 4;
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int s = s0 + n * join;
      const bool in = grp < join && e < quads && (kFull || d < D) && s < S;
      z[n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                           parts, in ? (s * (int)part + h * D + d) * 4 : (int)kOutOfRange, 0,
                                           kPolicyCoherent));
    }
  };
  u32x4 z[kBatch];
  fetch(z, join > 1 ? tid - grp * quads : tid, grp);
  float* const share = sh_o;                      // [head][S], at most kHeads * kMaxParts
  float* const sums = sh_o + kHeads * kMaxParts;  // [group][quads] of 4, at most kThreads * 4
  static_assert(kMaxParts <= 64, "a lane a part");
  for (int h = wave; h < nh; h += kWaves) {
    const int at = lane < S ? (lane * (int)part + D * kHeads + h) * 4 : (int)kOutOfRange;
    const float ms = coherent(at), ls = coherent(at + kHeads * 4);
    const float M = over_lanes(lane < S ? ms : -INFINITY, [](float u, float w) { return fmaxf(u, w); });
    const float Mu = M == -INFINITY ? 0.f : M;
    const float f = lane < S ? exp_((ms - Mu) * a.scale) : 0.f;
    const float W = over_lanes(f * ls, [](float u, float w) { return u + w; });
    if (lane < S) share[h * S + lane] = W == 0.f ? 0.f : f * inverse(W);
    if (lane == 0 && (a.lse || a.shares || kFused)) {
      const float z = W == 0.f ? -INFINITY : fmaf(Mu, a.scale, log_(W));
      const Share head = {Mu, fabsf(z) < INFINITY ? inverse(W) : 0.f};
      if (a.lse) a.lse[(long long)b * a.H + h0 + h] = z;
      if (a.shares) a.shares[(long long)b * a.H + h0 + h] = head;
      if (kFused) sh_share[h] = head;
    }
  }
  __syncthreads();
  if (kFused) add_weights();
  for (int e0 = 0; e0 < quads; e0 += kThreads) {
    const int e = join > 1 ? tid - grp * quads : e0 + tid;
    const int h = e / kQuads, d = e % kQuads * 4;
    const bool in = grp < join && e < quads && (kFull || d < D);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = grp; s0 < S; s0 += kBatch * join) {
      if (e0 > 0 || s0 >= join) fetch(z, e, s0);
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int s = s0 + n * join;
        if (in && s < S) {
          const float w = share[h * S + s];
          // A part of no weight adds nothing (its output may be infinite).
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] = w == 0.f ? o[c] : fmaf(w, __uint_as_float(z[n][c]), o[c]);
        }
      }
    }
    if (join > 1) {
      if (grp < join) *reinterpret_cast<f32x4*>(sums + tid * 4) = o;
      __syncthreads();
      if (grp != 0) return;
      for (int k = 1; k < join; ++k) o += *reinterpret_cast<const f32x4*>(sums + (k * quads + e) * 4);
    }
    if (in) {
      T* const to = static_cast<T*>(a.o) + b * a.os.b + (h0 + h) * a.os.h + d;
#pragma unroll
      for (int c = 0; c < 4; ++c) to[c] = (T)o[c];
    }
  }
}

// key_weights after the step: four keys a thread, the heads of the key-value head added in order.
__global__ __launch_bounds__(256) void add_weights_kernel(const float* __restrict__ scores,
                                                          const Share* __restrict__ shares,
                                                          const int* __restrict__ lens,
                                                          const int* __restrict__ table, long long table_stride,
                                                          float* weights, long long wb, long long wh,
                                                          long long n_pad, int H, int G, int P, int page,
                                                          int n_max, int append, float scale_log2) {
  const int b = blockIdx.z, kv = blockIdx.y;
  const int L = lens[b];
  if (L < 0 || L > n_max - append) return;
  const int j0 = (blockIdx.x * 256 + threadIdx.x) * 4;
  const long long first = (long long)b * H + kv * G;
  float* const to = weights + b * wb + kv * wh;
  if (j0 < L) {
    float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8  // (no branch on the head: the heads' loads go out together)
    for (int h = 0; h < G; ++h) {
      const Share head = shares[first + h];
      const f32x4 x = *reinterpret_cast<const f32x4*>(scores + (first + h) * n_pad + j0);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = add_weight(w[e], x[e], head, scale_log2);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j0 + e < L) to[j0 + e] += w[e];
  }
  if (append && j0 == 0 && (uint32_t)table[(long long)b * table_stride + L / page] < (uint32_t)P) {
    float w = 0.f;
#pragma unroll 8
    for (int h = 0; h < G; ++h) {
      w = add_weight(w, scores[(first + h + 1) * n_pad - kScoreTail], shares[first + h], scale_log2);
    }
    to[L] = w;
  }
}

// ---------------------------------------------------------------------------------------
// Host side.

// About kSlots workgroups a CU (a step of 4 sequences, 32 heads on 8, D = 128, 32768 rows: 80 us; with 1 102, with 4
// 83.5).
constexpr int kSlots = 2;
// A sequence by itself of at most kWhole rows, and a batch's of twice as many, is not divided (12 heads of 400 rows
// 6.4 us, divided 8.1; 1024 rows 8.5 divided, 9.7 not; 8 sequences of 1024, whose division takes the plan, 11.3
// divided, 10.2 not).
constexpr int kWhole = 512;
// The smallest part, in granules.  A unit of n granules in S parts takes a time of a n / S for its rows and b G S for
// writing and joining S outputs of G heads, least at parts n / S = sqrt(b / a) sqrt(n G): longer with G (28 heads on
// 4, D = 128, 8192 rows 14.6 us, with parts of 1 granule 18.4; 16 on 1, D = 64, 8192 rows 12.7 and 17.0, with parts
// of 8 14.3).
static int min_granules(int G) { return (int)lround(sqrt((double)std::min(kHeads, G))); }
// key_weights of a key-value head of at most kFusedRows rows and kFusedScores scores are added by the workgroup that
// ends it; more of them, and those of several units, by a kernel of their own, which takes the host another 2.5 us.
// One kernel against two: 32 heads on 8, D = 128, 4 sequences of 1000 rows 17.6 and 18.9 us, of 4000 20.4 and 21.2; 16
// heads on 1 of 1000 15.3 and 15.0; but 16 heads of 8000 rows 18.0 and 16.6, 32 on 8 heads of 8000 35.0 and 30.9.
constexpr long long kFusedRows = 6144, kFusedScores = 16384;
constexpr int kMaxCu = 1024;  // for the workspace's size, which does not depend on the device

static long long padded(long long n) { return (n + kGranule - 1) / kGranule * kGranule + kScoreTail; }

// Parts of the workspace for `wgs` workgroups and `units` units: arrival words, parts, shares, scores.
struct Layout {
  size_t part, shares, scores, bytes;
};
static Layout layout(long long units, long long wgs, long long bh, long long n_max, int D, bool weights) {
  Layout x;
  x.part = tfgfa::arrive_bytes(units);
  x.shares = x.part + ((size_t)wgs * part_floats(D) * 4 + 255) / 256 * 256;
  x.scores = x.shares + (weights ? ((size_t)bh * sizeof(Share) + 255) / 256 * 256 : 0);
  x.bytes = x.scores + (weights ? (size_t)bh * padded(n_max) * 4 : 0);
  return x;
}

// Workgroups that a division on a device of cu_count CUs may start: target a unit and one more a sequence's
// unit.  No division (target 0) where there are units enough, or where sequences are short.
static int choose_target(long long units, int B, long long n_max, int cu_count) {
  const long long per = units * B;
  // Sequences of like lengths take 1 to 2% longer divided from 4 units a CU on (128 of 8 heads of 4096 rows 188 us,
  // divided 189; 256 of 2048 180.4 and 183; 64 of 25 heads of 188 to 1500 64.6 and 66; below, 64 of 8 heads of 4096:
  // 67.7 and 65.7).  The lengths are not known here, and a very long one among that many pays for it: 128 sequences of
  // 8 heads, D = 128, one of 32768 rows and the others of 512, take 380 us, divided 75.  (Past 2^21 granules the
  // plan's quotients are not exact.)
  if (n_max <= (B == 1 ? kWhole : 2 * kWhole) || per >= (long long)kSlots * 2 * cu_count ||
      (n_max / kGranule + 1) * B >= 1 << 20)
    return 0;
  const long long target = std::max(1LL, (long long)kSlots * cu_count / units);
  if (B > 1) return (int)target;
  return (int)std::min<long long>(std::min<long long>(target, kMaxParts), (n_max + kGranule - 1) / kGranule);
}
static long long workgroups(long long units, int B, long long n_max, int target) {
  if (target == 0) return units * B;
  if (B == 1) return units * target;
  const long long most = (n_max + kGranule - 1) / kGranule;  // parts of a unit
  return units * std::min<long long>((long long)B * std::max(1LL, most), (long long)target + B);
}

static bool sizes_ok(int B, int H, int Hkv, int page, int M, int D) {
  if (B < 0 || H < 0 || Hkv < 0 || page < 1 || M < 0) return false;
  if (Hkv == 0 ? H != 0 : H % Hkv != 0) return false;
  return true;
}

// Granules of the whole batch and workgroups are counted in 32 bits; so are key indexes, with room for the blocks that
// a loop looks ahead.
static bool too_large(long long units, int B, int H, long long n_max) {
  return n_max > INT32_MAX - 128 * kMaxParts * kGranule || B > 65535 || units >= 1 << 20 ||
         (long long)B * H > INT32_MAX || units * B > INT32_MAX;
}

template <class T, int kDV, bool kFull>
static void launch_full(const First& f, const Args& a, unsigned wgs, hipStream_t stream) {
  const dim3 grid = f.target ? dim3(wgs) : dim3(f.units, f.B);
#define TFGFA_PAGED_(kSpan, kDivide, kFused)                                                                     \
  hipLaunchKernelGGL((paged_kernel<T, kDV, kFull, kSpan, kDivide, kFused>), grid, dim3(kThreads), 0, stream, f.table, \
                     f.lens, f.table_stride, static_cast<const T*>(f.q), f.n_max, f.div_m, f.div_s, f.target, f.units, \
                     f.B, a)
#define TFGFA_PAGED(kSpan)                                           \
  do {                                                               \
    if (a.weights && f.target) TFGFA_PAGED_(kSpan, true, true);      \
    else if (a.weights) TFGFA_PAGED_(kSpan, false, true);            \
    else if (f.target) TFGFA_PAGED_(kSpan, true, false);             \
    else TFGFA_PAGED_(kSpan, false, false);                          \
  } while (0)
  if (a.page % kTile == 0)
    TFGFA_PAGED(kTile);
  else
    TFGFA_PAGED(1);
#undef TFGFA_PAGED
#undef TFGFA_PAGED_
}
template <class T>
static void launch(const First& f, const Args& a, unsigned wgs, hipStream_t stream) {
  if (a.D == 64)
    launch_full<T, 4, true>(f, a, wgs, stream);
  else if (a.D < 64)
    launch_full<T, 4, false>(f, a, wgs, stream);
  else if (a.D == 128)
    launch_full<T, 8, true>(f, a, wgs, stream);
  else
    launch_full<T, 8, false>(f, a, wgs, stream);
}

}  // namespace tfgfa_paged

extern "C" size_t tfserve_decode_paged_workspace(int B, int H, int H_kv, int page, int M, int D,
                                                 int with_weights) {
  using namespace tfgfa_paged;
  if (!sizes_ok(B, H, H_kv, page, M, D) || D < 8 || D > kMaxD || (D & 7)) return 0;
  if (B == 0 || H == 0 || M == 0) return 0;
  const long long n_max = (long long)M * page, tiles = (H / H_kv + kHeads - 1) / kHeads;
  const long long units = H_kv * tiles;
  if (too_large(units, B, H, n_max)) return 0;
  long long wgs = 0;  // the most that any device of up to kMaxCu CUs starts
  const int target = choose_target(units, B, n_max, kMaxCu);
  if (target) wgs = workgroups(units, B, n_max, target);
  if (wgs == 0 && !with_weights) return 0;
  return layout(units * B, wgs, (long long)B * H, n_max, D, with_weights != 0).bytes;
}

extern "C" int tfserve_decode_paged(
    const void* q, const int64_t* q_strides, void* k_pages, const int64_t* k_strides, void* v_pages,
    const int64_t* v_strides, const int* page_table, int64_t table_stride, const int* cache_seqlens,
    const void* k_new, const int64_t* k_new_strides, const void* v_new, const int64_t* v_new_strides, void* o,
    const int64_t* o_strides, float* lse, float* key_weights, const int64_t* weights_strides, int B, int H,
    int H_kv, int P, int page, int M, int D, int dtype, float softmax_scale, void* workspace,
    size_t workspace_bytes, void* hip_stream) {
  using namespace tfgfa_paged;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16) return TFGFA_ERR_DTYPE;
  if (!sizes_ok(B, H, H_kv, page, M, D) || P < 0) return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7)) return TFGFA_ERR_HEAD_DIM;
  if (!(softmax_scale > 0.f) || !isfinite(softmax_scale)) return TFGFA_ERR_SCALE;
  if ((k_new == nullptr) != (v_new == nullptr)) return TFGFA_ERR_NULL_POINTER;
  const bool append = k_new != nullptr;
  if (B == 0 || H == 0) return TFGFA_OK;
  if (P == 0) return TFGFA_ERR_BAD_SHAPE;
  const long long n_max = (long long)M * page;
  Args a = {};
  First f = {};
  a.tiles = (H / H_kv + kHeads - 1) / kHeads;
  const long long units = (long long)H_kv * a.tiles;
  if (too_large(units, B, H, n_max)) return TFGFA_ERR_TOO_LARGE;
  if (!q_strides || !k_strides || !v_strides || !o_strides) return TFGFA_ERR_NULL_POINTER;
  if (append && (!k_new_strides || !v_new_strides)) return TFGFA_ERR_NULL_POINTER;
  if (!vecs_ok(q_strides, B, H, &a.qs) || !vecs_ok(o_strides, B, H, &a.os) ||
      !pages_ok(k_strides, P, H_kv, page, D, &a.ks) || !pages_ok(v_strides, P, H_kv, page, D, &a.vs))
    return TFGFA_ERR_STRIDE;
  // A block's rows, and a unit's queries, are one buffer of less than 2^30 bytes.
  if (a.ks.n >= (1 << 30) / kBlock || a.vs.n >= (1 << 30) / kBlock || 2 * a.qs.h >= (1 << 30) / kHeads)
    return TFGFA_ERR_TOO_LARGE;
  if (append && (!vecs_ok(k_new_strides, B, H_kv, &a.kns) || !vecs_ok(v_new_strides, B, H_kv, &a.vns)))
    return TFGFA_ERR_STRIDE;
  if (!apart(a.os.b, B, a.os.h, H, D)) return TFGFA_ERR_STRIDE;
  if (append && (!pages_apart(a.ks, P, H_kv, page, D) || !pages_apart(a.vs, P, H_kv, page, D))) return TFGFA_ERR_STRIDE;
  if (B > 1 && table_stride < 0) return TFGFA_ERR_STRIDE;
  if (!q || !k_pages || !v_pages || !o || !cache_seqlens || (!page_table && M > 0)) return TFGFA_ERR_NULL_POINTER;
  if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o | (uintptr_t)k_new |
       (uintptr_t)v_new | (uintptr_t)workspace) & 15u)
    return TFGFA_ERR_ALIGNMENT;
  if (((uintptr_t)lse | (uintptr_t)page_table | (uintptr_t)cache_seqlens | (uintptr_t)key_weights) & 3u)
    return TFGFA_ERR_ALIGNMENT;
  long long wb = 0, wh = 0;
  if (key_weights) {
    if (!weights_strides) return TFGFA_ERR_NULL_POINTER;
    wb = weights_strides[0], wh = weights_strides[1];
    if (!apart(wb, B, wh, H_kv, n_max)) return TFGFA_ERR_STRIDE;
    if (H_kv > 65535) return TFGFA_ERR_TOO_LARGE;
  }

  int cu = 0;
  const int st = tfgfa_device_info(&cu, nullptr, nullptr, 0);
  if (st != TFGFA_OK) return st;
  const bool weights = key_weights != nullptr && n_max > 0;
  f.target = choose_target(units, B, n_max, std::min(cu, kMaxCu));
  long long wgs = workgroups(units, B, n_max, f.target);
  Layout lay = layout(units * B, f.target ? wgs : 0, (long long)B * H, n_max, D, weights);
  if (lay.bytes > (workspace ? workspace_bytes : 0)) {
    if (weights) return TFGFA_ERR_SCRATCH;
    // Without a workspace that holds the division, each unit is one workgroup's.
    f.target = 0;
    wgs = workgroups(units, B, n_max, 0);
  }
  if (wgs > INT32_MAX) return TFGFA_ERR_TOO_LARGE;
  char* const ws = static_cast<char*>(workspace);
  f.table = page_table, f.table_stride = B > 1 ? table_stride : 0, f.lens = cache_seqlens, f.q = q;
  f.n_max = (int)n_max, f.units = (int)units, f.B = B;
  a.k = static_cast<char*>(k_pages), a.v = static_cast<char*>(v_pages);
  a.kn = k_new, a.vn = v_new, a.o = o, a.lse = lse;
  a.arrive = ws;
  a.part = ws ? reinterpret_cast<float*>(ws + lay.part) : nullptr;
  const bool fused = weights && a.tiles == 1 && n_max % 4 == 0 && n_max <= kFusedRows &&
                     n_max * (H / H_kv) <= kFusedScores;
  if (fused) a.weights = key_weights, a.wb = wb, a.wh = wh;
  a.shares = weights && !fused ? reinterpret_cast<Share*>(ws + lay.shares) : nullptr;
  a.scores = weights ? reinterpret_cast<float*>(ws + lay.scores) : nullptr;
  a.tag = f.target ? tfgfa::next_tag() : 0;
  a.n_pad = padded(n_max);
  a.scale = softmax_scale, a.scale_log2 = softmax_scale * kLog2e;
  const float slack = dtype == TFGFA_DTYPE_BF16 ? Elem<__bf16>::kSlack : Elem<_Float16>::kSlack;
  a.slack = std::min(slack / softmax_scale, 1e30f);
  a.H = H, a.G = H / H_kv, a.P = P, a.page = page, a.D = D;
  a.min_granules = min_granules(a.G);
  const tfgfa::Division by_page = tfgfa::division_by(page);
  f.div_m = by_page.m, f.div_s = by_page.s;
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (dtype == TFGFA_DTYPE_BF16)
    launch<__bf16>(f, a, (unsigned)wgs, stream);
  else
    launch<_Float16>(f, a, (unsigned)wgs, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && weights && !fused) {
    hipLaunchKernelGGL(add_weights_kernel, dim3((unsigned)((n_max + 1023) / 1024), H_kv, B), dim3(256), 0, stream,
                       a.scores, a.shares, cache_seqlens, page_table, f.table_stride, key_weights, wb, wh, a.n_pad,
                       H, a.G, P, page, (int)n_max, append ? 1 : 0, a.scale_log2);
    e = hipGetLastError();
  }
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
