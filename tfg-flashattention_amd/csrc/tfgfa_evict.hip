// tfgfa_evict.hip - eviction from a paged key-value cache by accumulated attention weight, MI355X (gfx950).
//
// Of the L rows of a (sequence, key-value head) the last `recent` stay, then those of the largest weight, ties to the
// lowest row, n = min(L, budget) in all; they are copied in their order to rows 0 .. n - 1 of other pages.
//
// select_kernel: one workgroup a (sequence, key-value head).  Bound: latency, a few passes over the head's weights,
// which stay in registers (up to 32768 rows; longer ones are read again in each pass).  Weights are ordered as 32-bit
// keys (the float's bits, flipped so that unsigned order is float order; NaN lowest).  The last key that is kept is
// found by its digits of 11, 11 and 10 bits: a histogram in LDS of the keys that share the digits found so far, and
// the digit at which the count from above reaches the number kept.  (The first digit is sign, exponent and two bits
// of the mantissa: weights spread over tens of its values, so that few of a wave's 64 additions meet.)  Then the rows
// above that key, and the first of those equal to it, are written behind one another: a wave's rows stand in row
// order, register by register, so places are counts of bits in ballots.
// copy_kernel: 16 bytes a thread and step, rows of K and V through both page tables.  Bound: HBM, 4D bytes read and
// 4D written a kept row.  Where a head has few rows to copy, the selecting workgroup copies them itself.
//
// Measured: 32 heads of up to 32768 rows, D = 128, cut to 4096: selection 23 us (32 of 256 CUs have work; 53% of the
// wave cycles in waits, for loads and at 17 barriers), copies 35 us, 3.9 TB/s of reads and writes (22, 6 TB/s, from
// the Infinity Cache); 16 sequences of 25 heads of up to 1024 rows cut to 512: 7.4 and 23 us (15.4); one sequence of
// 12 heads, 300 rows cut to 130, 7.5 us in one launch.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "tfgfa.h"
#include "tfgfa_layout.h"
#include "tfgfa_serving.h"

namespace tfgfa_evict {

using tfgfa::apart;
using tfgfa::Pages;
using tfgfa::pages_apart;
using tfgfa::pages_ok;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxD = 128;
constexpr int kBins = 2048;
constexpr int kMaxFused = kBins;  // rows that a selecting workgroup may copy itself (their list is in LDS)
// Rows with the first digit of the last one kept that a list holds, for the other digits (59.2 us at 32768 rows, 61.8
// with the registers gone through again).
constexpr int kCandidates = 4096;
constexpr int kFewRows = 4096;    // rows of a sequence that four weights a lane hold
constexpr int kMaxRows = 32768;   // rows of a sequence whose weights stay in registers
// rows * D of a head up to which the selecting workgroup copies them (12 heads, 130 rows: 7.6 us, with two kernels
// 9.7; 400 heads of 512 rows: 28.2 and 26.4).
constexpr int kFusedValues = 16384;
constexpr int kCopy = 4;          // rows of a thread of the copying kernel

struct Args {
  char* k;
  char* v;
  const int* table;
  const int* lens;
  const float* weights;
  const int* new_table;
  int* kept;
  float* out;
  Pages ks, vs;
  long long table_stride, new_stride, wb, wh, ob, oh;
  tfgfa::Division by_page;
  int Hkv, P, page, n_max, budget, recent, pieces, fused;
};

// Order of a weight as an unsigned number.
__device__ __forceinline__ uint32_t rank_key(float w) {
  const uint32_t x = __float_as_uint(w + 0.f);  // -0 as 0
  const uint32_t y = x >> 31 ? ~x : x | 0x80000000u;
  return w != w ? 0u : y;
}

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
  x = add_dpp<0x142, 0xA>(x);     // lane 15 of rows 0 and 2 to the row after
  return add_dpp<0x143, 0xC>(x);  // lane 31 to rows 2 and 3
}
// Bits of m below this lane's, and n.
__device__ __forceinline__ int below(unsigned long long m, int n) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, n));
}

__device__ __forceinline__ int page_of(const Args& a, int j) {
  return (int)(((unsigned long long)(uint32_t)j * a.by_page.m) >> a.by_page.s);
}

// Pages of the first n rows (n + page may pass 2^31).
__device__ __forceinline__ int pages_of(const Args& a, int n) { return n > 0 ? page_of(a, n - 1) + 1 : 0; }

// Rows i0, i0 + step, .. of the kept ones, 16-byte piece c of K and V, kUnroll at a time.  list(i): the row, or -1.
template <int kUnroll, class List>
__device__ __forceinline__ void copy_rows(const Args& a, int b, int kv, int i0, int step, int c, int n, List list) {
  const int* const from = a.table + b * a.table_stride;
  const int* const to = a.new_table + b * a.new_stride;
  for (; i0 < n; i0 += step * kUnroll) {
    u32x4 kx[kUnroll], vx[kUnroll];
    int j[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) j[u] = i0 + u * step < n ? list(i0 + u * step) : -1;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (j[u] >= 0) {
        const int at = page_of(a, j[u]);
        const long long p = from[at], r = j[u] - at * a.page;
        kx[u] = *reinterpret_cast<const u32x4*>(a.k + p * a.ks.p + kv * a.ks.h + r * a.ks.n + 16 * c);
        vx[u] = *reinterpret_cast<const u32x4*>(a.v + p * a.vs.p + kv * a.vs.h + r * a.vs.n + 16 * c);
      }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (j[u] >= 0) {
        const int i = i0 + u * step, at = page_of(a, i);
        const long long p = to[at], r = i - at * a.page;
        *reinterpret_cast<u32x4*>(a.k + p * a.ks.p + kv * a.ks.h + r * a.ks.n + 16 * c) = kx[u];
        *reinterpret_cast<u32x4*>(a.v + p * a.vs.p + kv * a.vs.h + r * a.vs.n + 16 * c) = vx[u];
      }
  }
}

// kW waves; kR weights a lane in registers (row of register r: (wave * kR + r) * 64 + lane), 0: read in each pass,
// wave by wave in the same order.
template <int kW, int kR>
__global__ __launch_bounds__(64 * kW) void select_kernel(const Args a) {
  constexpr int kThreads = 64 * kW, kEach = kBins / kThreads;
  constexpr bool kFuses = kR > 0 && kR <= 4;  // may copy the rows too
  constexpr bool kList = kR > 4;  // candidates of the second digit are put into a list where it holds them
  __shared__ int hist[kBins];
  __shared__ uint32_t list[kList ? kCandidates : 1];
  __shared__ int sh_sum[kW], sh_tie[kW];
  __shared__ int sh_digit, sh_above, sh_bad, sh_count;
  const int tid = threadIdx.x, lane = tid & 63, kv = blockIdx.x, b = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* const w = a.weights + b * a.wb + kv * a.wh;
  int* const kept = a.kept + ((long long)b * a.Hkv + kv) * a.budget;
  float* const out = a.out + b * a.ob + kv * a.oh;
  int L = a.lens[b];
  bool bad = L < 0 || L > a.n_max;
  if (bad) L = 0;
  const int n = min(L, a.budget);
  const bool every = L <= a.budget;
  // The rows from `old` on are protected; of those before it, `chosen` are kept.
  const int old = every ? 0 : L - min(L, a.recent), chosen = every ? 0 : n - (L - old);
  // This wave's rows: from `first` on.
  const int regs = kR > 0 ? kR : (L + kThreads - 1) / kThreads;
  const int first = wave * regs * 64;
  float x[kR > 0 ? kR : 1];
  uint32_t q[kR > 0 ? kR : 1];
  if constexpr (kR > 0) {
    // (Past the last row the buffer gives zeros.)
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(w), (short)0, 4 * L, 0x00020000);
#pragma unroll
    for (int r = 0; r < kR; ++r)
      x[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, (first + lane) * 4 + r * 256, 0, 0));
  }
  for (int c = tid; c < pages_of(a, L); c += kThreads)
    bad |= (uint32_t)a.table[b * a.table_stride + c] >= (uint32_t)a.P;
  for (int c = tid; c < pages_of(a, n); c += kThreads)
    bad |= (uint32_t)a.new_table[b * a.new_stride + c] >= (uint32_t)a.P;
  if (tid == 0) sh_bad = sh_count = 0;
  __syncthreads();
  if (bad) sh_bad = 1;
  if constexpr (kR > 0) {
#pragma unroll
    for (int r = 0; r < kR; ++r) q[r] = first + r * 64 + lane < old ? rank_key(x[r]) : 0u;
  }
  // f(key) for this wave's rows in order.  Rows that are not to be chosen from have the lowest key, which as the last one
  // in every order changes no count from above.
  auto rows = [&](auto f) {
    if constexpr (kR > 0) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        if (first + r * 64 >= old) break;
        f(q[r]);
      }
    } else {
      for (int r = 0; r < regs; ++r) {
        if (first + r * 64 >= old) break;
        const int j = first + r * 64 + lane;
        f(j < old ? rank_key(w[j]) : 0u);
      }
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int e = 0; e < kEach; ++e) hist[e * kThreads + tid] = 0;
    __syncthreads();
  };
  // One more of a digit, in the lanes that are in; a wave whose keys all have one digit (equal weights) adds them at
  // once.
  auto count = [&](bool in, int digit) {
    const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
    if (who == 0) return;
    const int lead = __builtin_amdgcn_readlane(digit, __builtin_ctzll(who));
    if (__builtin_amdgcn_ballot_w64(in && digit != lead) == 0) {
      if (lane == 0) atomicAdd(&hist[lead], __builtin_popcountll(who));
    } else if (in) {
      atomicAdd(&hist[digit], 1);
    }
  };
  // The chosen-th largest key, and how many of the keys equal to it are wanted.
  uint32_t key = 0;
  int want = chosen;
  // The digit at which the count of the histogram from above reaches `want`.
  auto find = [&](int shift) {
    __syncthreads();
    // Thread t: bins from kBins - 1 - t kEach down.
    int mine = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) mine += hist[kBins - 1 - tid * kEach - e];
    const int upto = scan64(mine);
    if (lane == 63) sh_sum[wave] = upto;
    __syncthreads();
    int above = upto - mine;
#pragma unroll
    for (int c = 0; c < kW; ++c) above += c < wave ? sh_sum[c] : 0;
    if (above < want && above + mine >= want) {
      int e = 0;
      for (; e < kEach - 1; ++e) {
        const int here = hist[kBins - 1 - tid * kEach - e];
        if (above + here >= want) break;
        above += here;
      }
      sh_digit = kBins - 1 - tid * kEach - e;
      sh_above = above;
    }
    __syncthreads();
    key |= (uint32_t)sh_digit << shift;
    want -= sh_above;
  };
  if (chosen > 0 && chosen < old) {
    clear();
    rows([&](uint32_t y) {
      const int digit = y >> 21;
      if (__builtin_amdgcn_ballot_w64(digit != __builtin_amdgcn_readfirstlane(digit)) != 0)
        atomicAdd(&hist[digit], 1);
      else if (lane == 0)
        atomicAdd(&hist[digit], 64);
    });
    find(21);
    const int same = hist[key >> 21];
    if (kList && same <= kCandidates) {
      __syncthreads();  // (the histogram has been read)
      int mine = 0;
      rows([&](uint32_t y) { mine += y >> 21 == key >> 21 ? 1 : 0; });
      const int upto = scan64(mine);
      int at = lane == 63 ? atomicAdd(&sh_count, upto) : 0;
      at = __builtin_amdgcn_readlane(at, 63) + upto - mine;
      rows([&](uint32_t y) {
        if (y >> 21 == key >> 21) list[at++ & (kCandidates - 1)] = y;
      });
#pragma unroll 1
      for (int shift = 10; shift >= 0; shift -= 10) {
        clear();
        for (int c = tid; c < (same + 63) / 64 * 64; c += kThreads) {
          const uint32_t y = c < same ? list[c] : 0u;
          const int top = shift == 10 ? 21 : 10;
          count(c < same && y >> top == key >> top, (y >> shift) & ((1 << (top - shift)) - 1));
        }
        find(shift);
      }
    } else {
#pragma unroll 1
      for (int shift = 10; shift >= 0; shift -= 10) {
        const int top = shift == 10 ? 21 : 10;
        __syncthreads();
        clear();
        rows([&](uint32_t y) { count(y >> top == key >> top, (y >> shift) & ((1 << (top - shift)) - 1)); });
        find(shift);
      }
    }
  } else {  // (none is chosen: chosen < old wherever the budget does not hold every row)
    key = 0xFFFFFFFEu;  // no weight's key is it or above it
  }
  __syncthreads();
  if (sh_bad) {
    for (int i = tid; i < a.budget; i += kThreads) {
      kept[i] = -1;
      out[i] = __uint_as_float(0x7FC00000u);
    }
    return;
  }
  if constexpr (kR > 0) {
    // Protected rows count as above every key, so that a kept row's place is the number of rows above the key before it,
    // and of the wanted ties.  Rows past the last have the lowest key: as ties they come after all that are wanted.
    auto key_of = [&](int r) {
      const int j = first + r * 64 + lane;
      return j >= old && j < L ? 0xFFFFFFFFu : q[r];
    };
    // Those of the waves before.  (Every weight is in a register by now: `out` may be `w`.)
    int taken = 0, ties = 0;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (first + r * 64 >= L) break;
      q[r] = key_of(r);
      taken += q[r] > key ? 1 : 0;
      ties += q[r] == key ? 1 : 0;
    }
    taken = scan64(taken), ties = scan64(ties);
    if (lane == 63) {
      sh_sum[wave] = taken;
      sh_tie[wave] = ties;
    }
    __syncthreads();
    taken = ties = 0;
#pragma unroll
    for (int c = 0; c < kW; ++c) {
      taken += c < wave ? sh_sum[c] : 0;
      ties += c < wave ? sh_tie[c] : 0;
    }
    taken = __builtin_amdgcn_readfirstlane(taken), ties = __builtin_amdgcn_readfirstlane(ties);
    const __amdgpu_buffer_rsrc_t to_kept = __builtin_amdgcn_make_buffer_rsrc(kept, (short)0, INT32_MAX, 0x00020000);
    const __amdgpu_buffer_rsrc_t to_out = __builtin_amdgcn_make_buffer_rsrc(out, (short)0, INT32_MAX, 0x00020000);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (first + r * 64 >= L) break;
      const unsigned long long mo = __builtin_amdgcn_ballot_w64(q[r] > key);
      const unsigned long long mt = __builtin_amdgcn_ballot_w64(q[r] == key);
      const int t = below(mt, ties), at = below(mo, taken) + min(t, want);
      if (q[r] > key || (q[r] == key && t < want)) {
        const int j = first + r * 64 + lane;
        __builtin_amdgcn_raw_buffer_store_b32((uint32_t)j, to_kept, at * 4, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[r]), to_out, at * 4, 0, 0);
        if (kFuses && a.fused) hist[at & (kBins - 1)] = j;
      }
      taken += __builtin_popcountll(mo);
      ties += __builtin_popcountll(mt);
    }
  } else {
    auto keep = [&](int at, int j, float y) { kept[at] = j, out[at] = y; };
    // `out` may be `w`: rows move down only, and a step's rows, of all waves, are read before any is written.
    int done = 0, seen = 0;
    for (int j0 = 0; j0 < L; j0 += kThreads) {
      const int j = j0 + tid;
      const bool in = j < old;
      const float y = j < L ? w[j] : 0.f;
      const uint32_t z = rank_key(y);
      const unsigned long long mo = __builtin_amdgcn_ballot_w64(in && z > key);
      const unsigned long long mt = __builtin_amdgcn_ballot_w64(in && z == key);
      __syncthreads();
      if (lane == 0) {
        sh_sum[wave] = __builtin_popcountll(mo);
        sh_tie[wave] = __builtin_popcountll(mt);
      }
      __syncthreads();
      int o = done, s = seen;
#pragma unroll
      for (int c = 0; c < kW; ++c) {
        o += c < wave ? sh_sum[c] : 0;
        s += c < wave ? sh_tie[c] : 0;
        done += sh_sum[c];
        seen += sh_tie[c];
      }
      const int t = below(mt, s);
      if (in && (z > key || (z == key && t < want))) keep(below(mo, o) + min(t, want), j, y);
      if (!in && j < L) keep(chosen + j - old, j, y);
    }
    __syncthreads();
  }
  for (int i = n + tid; i < a.budget; i += kThreads) {
    kept[i] = -1;
    out[i] = 0.f;
  }
  if (!kFuses || !a.fused) return;
  __syncthreads();
  const int per = kThreads / a.pieces, row = tid / a.pieces;
  if (row < per) copy_rows<4>(a, b, kv, row, per, tid - row * a.pieces, n, [&](int i) { return hist[i]; });
}

__global__ __launch_bounds__(256) void copy_kernel(const Args a) {
  const int kv = blockIdx.y, b = blockIdx.z;
  const int* const rows = a.kept + ((long long)b * a.Hkv + kv) * a.budget;
  const int per = 256 / a.pieces, row = threadIdx.x / a.pieces;
  const int i0 = blockIdx.x * per * kCopy;
  if (row < per)
    copy_rows<kCopy>(a, b, kv, i0 + row, per, threadIdx.x - row * a.pieces, min(a.budget, i0 + per * kCopy),
                     [&](int i) { return rows[i]; });
}

template <int kW, int kR>
static void launch(const Args& a, int B, hipStream_t stream) {
  hipLaunchKernelGGL((select_kernel<kW, kR>), dim3(a.Hkv, B), dim3(64 * kW), 0, stream, a);
}

}  // namespace tfgfa_evict

extern "C" int tfserve_evict(void* k_pages, const int64_t* k_strides, void* v_pages, const int64_t* v_strides,
                             const int* page_table, int64_t table_stride, const int* cache_seqlens,
                             const float* key_weights, const int64_t* weights_strides, const int* new_page_table,
                             int64_t new_table_stride, int* kept, float* weights_out,
                             const int64_t* weights_out_strides, int B, int H_kv, int P, int page, int M, int M_new,
                             int D, int budget, int recent, void* hip_stream) {
  using namespace tfgfa_evict;
  if (B < 0 || H_kv < 0 || P < 0 || page < 1 || M < 0 || M_new < 0 || budget < 0 || recent < 0 || recent > budget ||
      (long long)M_new * page < budget)
    return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7)) return TFGFA_ERR_HEAD_DIM;
  if (B == 0 || H_kv == 0 || budget == 0) return TFGFA_OK;
  if (P == 0) return TFGFA_ERR_BAD_SHAPE;
  const long long n_max = (long long)M * page;
  if (n_max > INT32_MAX - 65536 || (long long)M_new * page > INT32_MAX || budget > INT32_MAX - 65536 || B > 65535 ||
      H_kv > 65535)
    return TFGFA_ERR_TOO_LARGE;
  if (!k_strides || !v_strides || !weights_strides || !weights_out_strides) return TFGFA_ERR_NULL_POINTER;
  if (B > 1 && (table_stride < 0 || new_table_stride < M_new)) return TFGFA_ERR_STRIDE;
  Args a = {};
  if (!pages_ok(k_strides, P, H_kv, page, D, &a.ks) || !pages_ok(v_strides, P, H_kv, page, D, &a.vs) ||
      !pages_apart(a.ks, P, H_kv, page, D) || !pages_apart(a.vs, P, H_kv, page, D))
    return TFGFA_ERR_STRIDE;
  a.wb = B > 1 ? weights_strides[0] : 0, a.wh = H_kv > 1 ? weights_strides[1] : 0;
  a.ob = B > 1 ? weights_out_strides[0] : 0, a.oh = H_kv > 1 ? weights_out_strides[1] : 0;
  if (a.wb < 0 || a.wh < 0 || !apart(a.ob, B, a.oh, H_kv, budget))
    return TFGFA_ERR_STRIDE;
  if (!k_pages || !v_pages || !cache_seqlens || !new_page_table || !kept || !weights_out ||
      (M > 0 && (!page_table || !key_weights)))
    return TFGFA_ERR_NULL_POINTER;
  if (weights_out == key_weights && (a.wb != a.ob || a.wh != a.oh)) return TFGFA_ERR_STRIDE;
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15u) return TFGFA_ERR_ALIGNMENT;
  if (((uintptr_t)page_table | (uintptr_t)cache_seqlens | (uintptr_t)key_weights | (uintptr_t)new_page_table |
       (uintptr_t)kept | (uintptr_t)weights_out) & 3u)
    return TFGFA_ERR_ALIGNMENT;
  a.k = static_cast<char*>(k_pages), a.v = static_cast<char*>(v_pages);
  a.table = page_table, a.lens = cache_seqlens, a.weights = key_weights, a.new_table = new_page_table;
  a.kept = kept, a.out = weights_out;
  a.table_stride = B > 1 ? table_stride : 0, a.new_stride = B > 1 ? new_table_stride : 0;
  a.Hkv = H_kv, a.P = P, a.page = page, a.n_max = (int)n_max, a.budget = budget, a.recent = recent;
  a.by_page = tfgfa::division_by(page);
  a.pieces = D / 8;
  const int rows = std::min<long long>(budget, n_max);
  a.fused = n_max <= kFewRows && rows <= kMaxFused && (long long)rows * D <= kFusedValues;
  const hipStream_t stream = (hipStream_t)hip_stream;
  // The fewest registers that hold a head's weights, in waves that still leave other heads room (400 heads of 1024
  // rows: 26.4 us with 8 waves of 2 a lane, 26.8 with 4 of 4, 30.2 with 16 of 1; 12 heads: 8.8, 10.8 and 9.1; 32 heads
  // of 32768: 59.2 with 16 of 32, 63.3 with 8 of 64).
  if (n_max <= 1024)
    launch<8, 2>(a, B, stream);
  else if (n_max <= kFewRows)
    launch<16, 4>(a, B, stream);
  else if (n_max <= kMaxRows)
    launch<16, 32>(a, B, stream);
  else
    launch<16, 0>(a, B, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return -(int)e;
  if (!a.fused) {
    const int per = 256 / a.pieces * kCopy;
    hipLaunchKernelGGL(copy_kernel, dim3((rows + per - 1) / per, H_kv, B), dim3(256), 0, stream, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
