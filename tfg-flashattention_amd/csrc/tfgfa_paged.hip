// tfgfa_paged.hip - one decode step of attention over a paged key-value cache, MI355X (gfx950), bf16
// or fp16, head dims that are multiples of 8 up to 128, query heads sharing key-value heads.
//
// For each query head h of key-value head h' (G = H / H_kv of them):
//     x_j = scale q_h . k_j,   o_h = sum_j e^(x_j) v_j / sum_j e^(x_j),   lse_h = log sum_j e^(x_j)
// over the rows j < L of the sequence, row j being row j % page of page table[j / page].
//
// Bound: HBM.  Each K and V row is read once, 4D bytes for 4DG flops.  The 16 columns of a 16x16 matrix
// tile are the query heads of one key-value head, so that up to 16 of them cost what one does:
//   scores   S^T[key][head] = K Q^T     v_mfma_f32_16x16x32 (element type; products exact, fp32 sums)
//   output   O^T[dim][head] += V^T P^T  v_mfma_f32_16x16x4_f32, P and V in fp32
// The scores leave the first product with lane (g = lane / 16, i = lane % 16) holding keys 4g .. 4g + 3 of
// head i.  The second product takes, per instruction, one key of each g: its B operand is such a register
// as it stands, and its A operand is one dim of that key's V row per lane, i.e. the row in its natural
// order (lane i: kDV neighbouring dims, one per instruction).  So neither P nor V is moved between
// lanes, and P is not rounded.  The fp32 matrix rate (256 flops a CU and cycle) is 3 times what the
// bytes of V ask for at HBM speed.
//
// Division of the work.  A unit is a (sequence, key-value head, 16 query heads).  The lengths are known on
// the device only, so every workgroup works the division out from them (plan, below): one chunk length C for
// all units, with about `target` workgroups in all; a unit of more than C rows is divided over
// several workgroups.  Each leaves its part (normalised output and log-sum-exp) in the workspace, and the
// one that arrives last joins them (arrival words and memory order as in tfgfa_decode.hip).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "tfgfa.h"
#include "tfgfa_arrive.h"
#include "tfgfa_layout.h"
#include "tfgfa_serving.h"

namespace tfgfa_paged {

using tfgfa::apart;
using tfgfa::Pages;
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
constexpr int kTiles = 2;                     // tiles of a wave's block
constexpr int kBlock = kTile * kTiles;        // keys of a wave's block
constexpr int kGranule = kWaves * kBlock;     // keys of a workgroup's block
constexpr int kMaxParts = 1024;               // workgroups of a unit (the arrival count has 16 bits)

template <class T>
struct Elem;
template <>
struct Elem<__bf16> {
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                   c, 0, 0, 0);
  }
  static __device__ __forceinline__ float lo(uint32_t x) { return __uint_as_float(x << 16); }
  static __device__ __forceinline__ float hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
};
template <>
struct Elem<_Float16> {
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                  0, 0, 0);
  }
  static __device__ __forceinline__ float lo(uint32_t x) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(x & 0xffffu));
  }
  static __device__ __forceinline__ float hi(uint32_t x) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(x >> 16));
  }
};

// e^x as 2^(x log2 e), the difference of two scores taken first: scores up to the largest float keep their place.
// v_exp_f32: results below 2^-126 are 0.
__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ float log_(float x) { return log2f(x) * kLn2; }

struct Args {
  const void* q;
  const char* k;
  const char* v;
  const int* table;
  const int* lens;
  const void* kn;
  const void* vn;
  void* o;
  float* lse;       // natural log, or null
  char* arrive;
  float* part;      // per workgroup of a divided unit: [head][D] outputs, then [head] LSE
  float* lse_ws;    // (B, H) LSE for the weights, or null
  float* scores;    // (B, H, n_pad) scores, or null
  u64 tag;
  long long table_stride;
  Pages ks, vs;
  Vecs qs, os, kns, vns;
  long long n_pad;
  float scale;
  int B, H, Hkv, G, P, page, n_max, D;
  int tiles;        // 16-head tiles of a key-value head
  int units;        // Hkv * tiles: units of one sequence
  int target;       // workgroups per unit of a sequence that the division aims at, in all sequences (0: no division)
  int min_granules; // smallest chunk
  uint32_t div_m;   // j / page = j * div_m >> div_s, j < 2^31
  int div_s;
};

__device__ __forceinline__ uint32_t div_page(const Args& a, uint32_t j) {
  return (uint32_t)(((u64)j * a.div_m) >> a.div_s);
}

// Sum of x over the lanes up to and with this one.
__device__ __forceinline__ int scan64(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

struct Piece {
  int b, unit, s, S;  // sequence, unit of it, part s of S
  int first;          // the unit's first workgroup
  int chunk;          // granules of a part
};

__device__ __forceinline__ int row_length(const Args& a, int n, bool append, bool* valid) {
  const bool ok = n >= 0 && n <= a.n_max - (append ? 1 : 0);
  *valid = ok;
  return ok ? n + (append ? 1 : 0) : 0;
}

// Granules of a sequence, at least one (a workgroup has to write the empty row).
__device__ __forceinline__ int granules(const Args& a, int b, bool append) {
  if (b >= a.B) return 0;
  bool valid;
  const int n = row_length(a, a.lens[b], append, &valid);
  return max(1, (n + kGranule - 1) / kGranule);
}

// The piece of work of workgroup w: with C = ceil(all granules / target) granules to a chunk, sequence b
// takes ceil(granules_b / C) workgroups for each of its units, in the order of (sequence, unit, part).
// Every wave of every workgroup computes it alike; false where no work is left.
__device__ __forceinline__ bool plan(const Args& a, int w, int lane, bool append, Piece* out) {
  int C = INT32_MAX;
  if (a.target > 0) {
    int total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int mine = granules(a, b0 + lane, append);
      total += __builtin_amdgcn_readlane(scan64(mine, lane), 63);
    }
    C = max(a.min_granules, (total + a.target - 1) / a.target);
    C = max(C, (a.n_max + kGranule * kMaxParts - 1) / (kGranule * kMaxParts));
  }
  int before = 0;  // parts of one unit in the sequences before
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int g = granules(a, b0 + lane, append);
    const int S = g == 0 ? 0 : C == INT32_MAX ? 1 : (g + C - 1) / C;
    const int upto = before + scan64(S, lane);
    const u64 done = __builtin_amdgcn_ballot_w64((long long)upto * a.units <= w);
    const int at = __builtin_popcountll(done);
    if (at < 64 && b0 + at < a.B) {
      const int Sb = __builtin_amdgcn_readlane(S, at);
      const int first = (__builtin_amdgcn_readlane(upto, at) - Sb) * a.units;
      const int i = w - first;
      out->b = b0 + at;
      out->unit = i / Sb;
      out->s = i - out->unit * Sb;
      out->S = Sb;
      out->first = first + out->unit * Sb;
      out->chunk = C;
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// A block of a wave: kTiles tiles of 16 keys.  k: row i of the tile, dims 32p + 8g of piece p (the A operand
// of the scores); v: per register r of a tile's scores the row 4g + r, dims kDV i ...
template <int kDV>
struct KV {
  u32x4 k[kTiles][kDV / 2];
  uint32_t v[kTiles][4][kDV / 2];
  bool bad[kTiles];
};

template <int kDV>
__device__ __forceinline__ void load_v(uint32_t (&x)[kDV / 2], const char* p) {
  if constexpr (kDV == 8) {
    const u32x4 y = *reinterpret_cast<const u32x4*>(p);
    x[0] = y[0], x[1] = y[1], x[2] = y[2], x[3] = y[3];
  } else {
    const u32x2 y = *reinterpret_cast<const u32x2*>(p);
    x[0] = y[0], x[1] = y[1];
  }
}

// kDV: dims of a lane in V, 4 (D <= 64) or 8.  kFull: D == 16 kDV.  kAligned: pages are whole tiles, so that the
// keys of a tile are in one page.
template <class T, int kDV, bool kFull, bool kAligned>
__global__ __launch_bounds__(kThreads, 2) void paged_kernel(const Args a) {
  constexpr int kDP = kDV / 2;          // pieces of 32 dims
  constexpr int kDm = 16 * kDV;
  __shared__ float sh_o[kWaves][kHeads][kDm + 4];
  __shared__ float sh_m[kWaves][kHeads], sh_l[kWaves][kHeads];
  __shared__ int sh_last;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, i = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool append = a.kn != nullptr;
  Piece pc;
  if (!plan(a, blockIdx.x, lane, append, &pc)) return;
  const int b = __builtin_amdgcn_readfirstlane(pc.b), unit = __builtin_amdgcn_readfirstlane(pc.unit);
  const int kv = unit / a.tiles, tile = unit - kv * a.tiles;
  const int h0 = kv * a.G + tile * kHeads;               // first query head
  const int nh = min(kHeads, a.G - tile * kHeads);       // query heads of the unit
  const int Lc = a.lens[b];
  bool valid;
  const int L = row_length(a, Lc, append, &valid);
  const int Lr = append ? L - 1 : L;  // rows that are in the cache (-1: an invalid appending row)
  const int D = a.D;
  const int c0 = pc.S > 1 ? pc.s * pc.chunk * kGranule : 0;
  const int c1 = pc.S > 1 ? min(L, c0 + pc.chunk * kGranule) : L;
  const int* const row = a.table + (long long)b * a.table_stride;
  u64* const aw = reinterpret_cast<u64*>(a.arrive + ((long long)b * a.units + unit) * tfgfa::kArriveStride);
  u64 aw_start = 0;
  if (pc.S > 1 && wave == 0)
    aw_start = __hip_atomic_load(aw, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // Queries: the B operand, head i, zero past the unit's heads and past D.
  u32x4 qf[kDP];
#pragma unroll
  for (int p = 0; p < kDP; ++p) {
    qf[p] = u32x4{0, 0, 0, 0};
    if (i < nh && (kFull || 32 * p + 8 * g < D))
      qf[p] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.q) + b * a.qs.b + (h0 + i) * a.qs.h +
                                              32 * p + 8 * g);
  }

  const char* const kh = a.k + kv * a.ks.h;
  const char* const vh = a.v + kv * a.vs.h;
  const char* const kn = append ? reinterpret_cast<const char*>(static_cast<const T*>(a.kn) + b * a.kns.b +
                                                                kv * a.kns.h)
                                : nullptr;
  const char* const vn = append ? reinterpret_cast<const char*>(static_cast<const T*>(a.vn) + b * a.vns.b +
                                                                kv * a.vns.h)
                                : nullptr;

  float m = -INFINITY, l = 0.f;
  f32x4 acc[kDV];
#pragma unroll
  for (int j = 0; j < kDV; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int kb = c0 + wave * kBlock; kb < c1; kb += kGranule) {
    KV<kDV> x;
    const bool tail = kb + kBlock > Lr;  // holds the new row, or rows past the length
    float s[kTiles][4];
    // Loads.  Rows at or past L of a page are inside it and may be read; their values are dropped below.
    // A tile of nothing but such rows is left out: the table need not have a page for it.
    bool new_ok = false;
    long long new_row_k = 0, new_row_v = 0;
    if constexpr (kAligned) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int key0 = kb + t * kTile;
        x.bad[t] = false;
        if (key0 < c1) {
          const uint32_t at = div_page(a, key0);
          int pid = __builtin_amdgcn_readfirstlane(row[at]);
          x.bad[t] = (uint32_t)pid >= (uint32_t)a.P;
          pid = x.bad[t] ? 0 : pid;
          const int off = key0 - at * a.page;
          const char* kp = kh + pid * a.ks.p + (off + i) * a.ks.n + 16 * g;
          if (tail && append && key0 + i == Lr) {
            new_ok = !x.bad[t];
            new_row_k = kp - kh;
            kp = kn + 16 * g;
          }
#pragma unroll
          for (int p = 0; p < kDP; ++p)
            x.k[t][p] = kFull || 32 * p + 8 * g < D ? *reinterpret_cast<const u32x4*>(kp + 64 * p)
                                                    : u32x4{0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const char* vp = vh + pid * a.vs.p + (off + 4 * g + r) * a.vs.n + 2 * kDV * i;
            if (tail && append && key0 + 4 * g + r == Lr) {
              new_row_v = vp - vh;
              vp = vn + 2 * kDV * i;
            }
#pragma unroll
            for (int e = 0; e < kDP; ++e) x.v[t][r][e] = 0;
            if (kFull || kDV * i < D) load_v<kDV>(x.v[t][r], vp);
          }
        } else {
#pragma unroll
          for (int p = 0; p < kDP; ++p) x.k[t][p] = u32x4{0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < kDP; ++e) x.v[t][r][e] = 0;
        }
      }
    } else {
      // Lane l looks up key kb + l % 32; the rows of the lanes' keys come from there.
      const int key = kb + (lane & (kBlock - 1));
      const uint32_t at = div_page(a, key);
      int pid = -1, off = 0;
      if (key < c1) {
        pid = row[at];
        off = key - at * a.page;
        if ((uint32_t)pid >= (uint32_t)a.P) pid = -1;
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int key0 = kb + t * kTile;
        x.bad[t] = false;
        const int kp_id = __shfl(pid, t * kTile + i), kp_off = __shfl(off, t * kTile + i);
        const bool is_new = append && key0 + i == Lr;
        const char* kp = kh + max(kp_id, 0) * a.ks.p + kp_off * a.ks.n + 16 * g;
        if (is_new) {
          new_ok = kp_id >= 0;
          new_row_k = kp - kh;
          kp = kn + 16 * g;
        }
#pragma unroll
        for (int p = 0; p < kDP; ++p)
          x.k[t][p] = key0 + i < c1 && (kp_id >= 0 || is_new) && (kFull || 32 * p + 8 * g < D)
                          ? *reinterpret_cast<const u32x4*>(kp + 64 * p)
                          : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k2 = key0 + 4 * g + r;
          const int id = __shfl(pid, t * kTile + 4 * g + r), of = __shfl(off, t * kTile + 4 * g + r);
          const char* vp = vh + max(id, 0) * a.vs.p + of * a.vs.n + 2 * kDV * i;
          const bool new_v = append && k2 == Lr;
          if (new_v) {
            new_row_v = vp - vh;
            vp = vn + 2 * kDV * i;
          }
          // A key of a bad page: the score below is NaN (marked by s here).
          s[t][r] = k2 < c1 && id < 0 ? __uint_as_float(0x7FC00000u) : 0.f;
#pragma unroll
          for (int e = 0; e < kDP; ++e) x.v[t][r][e] = 0;
          if (k2 < c1 && (id >= 0 || new_v) && (kFull || kDV * i < D)) load_v<kDV>(x.v[t][r], vp);
        }
      }
    }

    // The new row goes to its page from the lanes that hold it, in the unit's first 16 heads only.
    if (tail && append && tile == 0 && kb <= Lr && Lr < kb + kBlock) {
      const u64 who = __builtin_amdgcn_ballot_w64(new_ok);
      if (who != 0) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          if (kb + t * kTile + i == Lr)
#pragma unroll
            for (int p = 0; p < kDP; ++p)
              if (kFull || 32 * p + 8 * g < D)
                *reinterpret_cast<u32x4*>(const_cast<char*>(kh) + new_row_k + 64 * p) = x.k[t][p];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kb + t * kTile + 4 * g + r == Lr && (kFull || kDV * i < D)) {
              uint32_t* to = reinterpret_cast<uint32_t*>(const_cast<char*>(vh) + new_row_v);
#pragma unroll
              for (int e = 0; e < kDP; ++e) to[e] = x.v[t][r][e];
            }
        }
      }
    }

    // Scores; -inf past the length, NaN through a bad page.
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < kDP; ++p) c = Elem<T>::mfma(x.k[t][p], qf[p], c);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y = c[r] * a.scale;
        if constexpr (kAligned) {
          if (x.bad[t]) y = __uint_as_float(0x7FC00000u);
        } else {
          y += s[t][r];
        }
        if (tail) {
          const bool in = kb + t * kTile + 4 * g + r < L;
          y = in ? y : -INFINITY;
          if (!in)
#pragma unroll
            for (int e = 0; e < kDP; ++e) x.v[t][r][e] = 0;
        }
        s[t][r] = y;
      }
      if (a.scores != nullptr && i < nh && kb + t * kTile < c1)
        *reinterpret_cast<f32x4*>(a.scores + ((long long)b * a.H + h0 + i) * a.n_pad + kb + t * kTile + 4 * g) =
            f32x4{s[t][0], s[t][1], s[t][2], s[t][3]};
    }
    // Running maximum of each head over the wave's keys.
    float mb = s[0][0];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mb = fmaxf(mb, s[t][r]);
    mb = fmaxf(mb, __shfl_xor(mb, 16));
    mb = fmaxf(mb, __shfl_xor(mb, 32));
    if (__builtin_amdgcn_ballot_w64(mb > m)) {
      const float mn = fmaxf(m, mb);
      const float f = m == -INFINITY ? 0.f : exp_(m - mn);
      l *= f;
#pragma unroll
      for (int j = 0; j < kDV; ++j) acc[j] *= f;
      m = mn;
    }
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = exp_(s[t][r] - mu);
        l += p;
#pragma unroll
        for (int e = 0; e < kDP; ++e) {
          acc[2 * e] = __builtin_amdgcn_mfma_f32_16x16x4f32(Elem<T>::lo(x.v[t][r][e]), p, acc[2 * e], 0, 0, 0);
          acc[2 * e + 1] =
              __builtin_amdgcn_mfma_f32_16x16x4f32(Elem<T>::hi(x.v[t][r][e]), p, acc[2 * e + 1], 0, 0, 0);
        }
      }
  }
  if (pc.S > 1 && wave == 0 && lane == 0 && (aw_start >> tfgfa::kTagShift) != a.tag) {
    u64 expected = aw_start;
    __hip_atomic_compare_exchange_strong(aw, &expected, a.tag << tfgfa::kTagShift, __ATOMIC_RELAXED,
                                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }

  // Join the waves.  acc[j], register r of lane (g, i): dim kDV (4g + r) + j of head i.
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (i < nh) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < kDV; ++j) sh_o[wave][i][kDV * (4 * g + r) + j] = acc[j][r];
    if (g == 0) {
      sh_m[wave][i] = m;
      sh_l[wave][i] = l;
    }
  }
  __syncthreads();
  float* const mine = a.part + (long long)blockIdx.x * kHeads * (D + 1);
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
      const float f = exp_(sh_m[w][h] - Mu);
      lt = fmaf(f, sh_l[w][h], lt);
      ot = fmaf(f, sh_o[w][h][d], ot);
    }
    const float on = lt == 0.f ? 0.f : ot / lt;
    const float ls = lt == 0.f ? -INFINITY : Mu + log_(lt);
    if (pc.S == 1) {
      const float nan = __uint_as_float(0x7FC00000u);
      static_cast<T*>(a.o)[b * a.os.b + (h0 + h) * a.os.h + d] = (T)(valid ? on : nan);
      if (d == 0) {
        if (a.lse) a.lse[(long long)b * a.H + h0 + h] = valid ? ls : nan;
        if (a.lse_ws) a.lse_ws[(long long)b * a.H + h0 + h] = ls;
      }
    } else {
      __hip_atomic_store(mine + h * D + d, on, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0) __hip_atomic_store(mine + kHeads * D + h, ls, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (pc.S == 1) return;
  // The part is at the coherence point once its stores are acknowledged; then the arrival is counted.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const u64 old = __hip_atomic_fetch_add(aw, (u64)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int last = (old & ((1ull << tfgfa::kTagShift) - 1)) == (u64)(pc.S - 1);
    if (last) __hip_atomic_store(aw, (u64)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh_last = last;
  }
  __syncthreads();
  if (!sh_last) return;
  asm volatile("" ::: "memory");
  const long long step = (long long)kHeads * (D + 1);
  const float* const parts = a.part + pc.first * step;
  for (int e = tid; e < nh * kDm; e += kThreads) {
    const int h = e / kDm, d = e % kDm;
    if (!kFull && d >= D) continue;
    float M = -INFINITY, W = 0.f, o = 0.f;
    for (int s = 0; s < pc.S; ++s) {
      const float ls = __hip_atomic_load(parts + s * step + kHeads * D + h, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const float os = __hip_atomic_load(parts + s * step + h * D + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const float Mn = fmaxf(M, ls);
      const float Mu = Mn == -INFINITY ? 0.f : Mn;
      const float f = M == -INFINITY ? 0.f : exp_(M - Mu), w = exp_(ls - Mu);
      W = fmaf(W, f, w);
      o = fmaf(o, f, w * os);
      M = Mn;
    }
    const float ls = W == 0.f ? -INFINITY : M + log_(W);
    static_cast<T*>(a.o)[b * a.os.b + (h0 + h) * a.os.h + d] = (T)(W == 0.f ? 0.f : o / W);
    if (d == 0) {
      if (a.lse) a.lse[(long long)b * a.H + h0 + h] = ls;
      if (a.lse_ws) a.lse_ws[(long long)b * a.H + h0 + h] = ls;
    }
  }
}

// key_weights: four keys a thread, the heads of the key-value head added in order.
__global__ __launch_bounds__(256) void add_weights_kernel(const float* __restrict__ scores,
                                                          const float* __restrict__ lse_ws,
                                                          const int* __restrict__ lens,
                                                          const int* __restrict__ table, long long table_stride,
                                                          float* weights, long long wb, long long wh,
                                                          long long n_pad, int H, int G, int P, int page,
                                                          int n_max, int append) {
  const int b = blockIdx.z, kv = blockIdx.y;
  const int Lc = lens[b];
  if (Lc < 0 || Lc > n_max - append) return;
  const int L = Lc + append;
  const int j0 = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (j0 >= L) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  const long long first = (long long)b * H + kv * G;
  for (int h = 0; h < G; ++h) {
    const float z = lse_ws[first + h];
    if (!(fabsf(z) < INFINITY)) continue;
    const f32x4 x = *reinterpret_cast<const f32x4*>(scores + (first + h) * n_pad + j0);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] += exp_(x[e] - z);
  }
  float* const to = weights + b * wb + kv * wh;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = j0 + e;
    if (j < Lc)
      to[j] += w[e];
    else if (j < L && (uint32_t)table[(long long)b * table_stride + j / page] < (uint32_t)P)
      to[j] = w[e];
  }
}

// ---------------------------------------------------------------------------------------
// Host side.

// A workgroup's chunk: about kSlots workgroups a CU, no chunk below kMinGranules.
constexpr int kSlots = 2;
constexpr int kMinGranules = 2;
constexpr int kMaxCu = 1024;  // for the workspace's size, which does not depend on the device

static long long padded(long long n) { return (n + kGranule - 1) / kGranule * kGranule; }

// Parts of the workspace for `wgs` workgroups and `units` units: arrival words, parts, LSE, scores.
struct Layout {
  size_t part, lse_ws, scores, bytes;
};
static Layout layout(long long units, long long wgs, long long bh, long long n_max, int D, bool weights) {
  Layout x;
  x.part = tfgfa::arrive_bytes(units);
  x.lse_ws = x.part + ((size_t)wgs * kHeads * (D + 1) * 4 + 255) / 256 * 256;
  x.scores = x.lse_ws + (weights ? ((size_t)bh * 4 + 255) / 256 * 256 : 0);
  x.bytes = x.scores + (weights ? (size_t)bh * padded(n_max) * 4 : 0);
  return x;
}

// Workgroups that a division on a device of cu_count CUs may start: target a unit and one more a sequence's
// unit.  No division (target 0) where there are units enough, or where sequences are short.
static int choose_target(long long units, int B, long long n_max, int cu_count) {
  const long long per = units * B;
  if (n_max <= kMinGranules * kGranule || per >= (long long)kSlots * 2 * cu_count) return 0;
  return (int)std::max(1LL, (long long)kSlots * cu_count / units);
}
static long long workgroups(long long units, int B, long long n_max, int target) {
  if (target == 0) return units * B;
  const long long most = (n_max + kGranule - 1) / kGranule;  // parts of a unit
  return units * std::min<long long>((long long)B * std::max(1LL, most), (long long)target + B);
}

static bool sizes_ok(int B, int H, int Hkv, int page, int M, int D) {
  if (B < 0 || H < 0 || Hkv < 0 || page < 1 || M < 0) return false;
  if (Hkv == 0 ? H != 0 : H % Hkv != 0) return false;
  return true;
}

template <class T>
static void launch(const Args& a, unsigned grid, hipStream_t stream) {
  const bool aligned = a.page % kTile == 0;
#define TFGFA_PAGED(kDV, kFull, kAligned) \
  hipLaunchKernelGGL((paged_kernel<T, kDV, kFull, kAligned>), dim3(grid), dim3(kThreads), 0, stream, a)
  if (a.D == 64) {
    if (aligned) TFGFA_PAGED(4, true, true);
    else TFGFA_PAGED(4, true, false);
  } else if (a.D < 64) {
    if (aligned) TFGFA_PAGED(4, false, true);
    else TFGFA_PAGED(4, false, false);
  } else if (a.D == 128) {
    if (aligned) TFGFA_PAGED(8, true, true);
    else TFGFA_PAGED(8, true, false);
  } else {
    if (aligned) TFGFA_PAGED(8, false, true);
    else TFGFA_PAGED(8, false, false);
  }
#undef TFGFA_PAGED
}

}  // namespace tfgfa_paged

extern "C" size_t tfserve_decode_paged_workspace(int B, int H, int H_kv, int page, int M, int D,
                                                 int with_weights) {
  using namespace tfgfa_paged;
  if (!sizes_ok(B, H, H_kv, page, M, D) || D < 8 || D > kMaxD || (D & 7)) return 0;
  if (B == 0 || H == 0 || M == 0) return 0;
  const long long n_max = (long long)M * page, tiles = (H / H_kv + kHeads - 1) / kHeads;
  const long long units = H_kv * tiles;
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
  a.tiles = (H / H_kv + kHeads - 1) / kHeads;
  const long long units = (long long)H_kv * a.tiles;
  // Granules of the whole batch and workgroups are counted in 32 bits; so are key indexes, with room for a block.
  if (n_max > INT32_MAX - kGranule || units * B > INT32_MAX / 4 || (long long)B * H > INT32_MAX ||
      (n_max / kGranule + 1) * B > INT32_MAX)
    return TFGFA_ERR_TOO_LARGE;
  if (!q_strides || !k_strides || !v_strides || !o_strides) return TFGFA_ERR_NULL_POINTER;
  if (append && (!k_new_strides || !v_new_strides)) return TFGFA_ERR_NULL_POINTER;
  if (!vecs_ok(q_strides, B, H, &a.qs) || !vecs_ok(o_strides, B, H, &a.os) ||
      !pages_ok(k_strides, P, H_kv, page, D, &a.ks) || !pages_ok(v_strides, P, H_kv, page, D, &a.vs))
    return TFGFA_ERR_STRIDE;
  if (append && (!vecs_ok(k_new_strides, B, H_kv, &a.kns) || !vecs_ok(v_new_strides, B, H_kv, &a.vns)))
    return TFGFA_ERR_STRIDE;
  if (!apart(a.os.b, B, a.os.h, H, D)) return TFGFA_ERR_STRIDE;
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
    if (B > 65535 || H_kv > 65535) return TFGFA_ERR_TOO_LARGE;
  }

  int cu = 0;
  const int st = tfgfa_device_info(&cu, nullptr, nullptr, 0);
  if (st != TFGFA_OK) return st;
  const bool weights = key_weights != nullptr && n_max > 0;
  a.target = choose_target(units, B, n_max, std::min(cu, kMaxCu));
  long long wgs = workgroups(units, B, n_max, a.target);
  Layout lay = layout(units * B, a.target ? wgs : 0, (long long)B * H, n_max, D, weights);
  if (lay.bytes > (workspace ? workspace_bytes : 0)) {
    if (weights) return TFGFA_ERR_SCRATCH;
    // Without a workspace that holds the division, each unit is one workgroup's.
    a.target = 0;
    wgs = workgroups(units, B, n_max, 0);
  }
  if (wgs > INT32_MAX) return TFGFA_ERR_TOO_LARGE;
  char* const ws = static_cast<char*>(workspace);
  a.q = q, a.k = static_cast<char*>(k_pages), a.v = static_cast<char*>(v_pages);
  a.table = page_table, a.table_stride = B > 1 ? table_stride : 0, a.lens = cache_seqlens;
  a.kn = k_new, a.vn = v_new, a.o = o, a.lse = lse;
  a.arrive = ws;
  a.part = ws ? reinterpret_cast<float*>(ws + lay.part) : nullptr;
  a.lse_ws = weights ? reinterpret_cast<float*>(ws + lay.lse_ws) : nullptr;
  a.scores = weights ? reinterpret_cast<float*>(ws + lay.scores) : nullptr;
  a.tag = a.target ? tfgfa::next_tag() : 0;
  a.n_pad = padded(n_max);
  a.scale = softmax_scale;
  a.B = B, a.H = H, a.Hkv = H_kv, a.G = H / H_kv, a.P = P, a.page = page, a.n_max = (int)n_max, a.D = D;
  a.units = (int)units;
  a.min_granules = kMinGranules;
  // j / page by a product: with 2^(l-1) < page <= 2^l and m = floor(2^(31+l) / page) + 1 the error j (m page -
  // 2^(31+l)) / 2^(31+l) is below 1 / page for j < 2^31, and m < 2^32.
  int lg = 0;
  while ((1LL << lg) < page) ++lg;
  a.div_m = (uint32_t)((1ULL << (31 + lg)) / (uint64_t)page + 1);
  a.div_s = 31 + lg;
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (dtype == TFGFA_DTYPE_BF16)
    launch<__bf16>(a, (unsigned)wgs, stream);
  else
    launch<_Float16>(a, (unsigned)wgs, stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && weights) {
    hipLaunchKernelGGL(add_weights_kernel, dim3((unsigned)((n_max + 1023) / 1024), H_kv, B), dim3(256), 0, stream,
                       a.scores, a.lse_ws, cache_seqlens, page_table, a.table_stride, key_weights, wb, wh, a.n_pad,
                       H, a.G, P, page, (int)n_max, append ? 1 : 0);
    e = hipGetLastError();
  }
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
