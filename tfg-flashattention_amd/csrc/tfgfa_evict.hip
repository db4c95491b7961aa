// tfgfa_evict.hip - eviction from a paged key-value cache by accumulated attention weight, MI355X (gfx950).
//
// Of the L rows of a (sequence, key-value head) the last `recent` stay, then those of the largest weight, ties to the
// lowest row, n = min(L, budget) in all; they are copied in their order to rows 0 .. n - 1 of other pages.
//
// select_kernel: one workgroup a (sequence, key-value head).  Weights are ordered as 32-bit keys (the float's
// bits, flipped so that unsigned order is float order; NaN lowest, protected rows highest).  The n-th largest key is
// found digit by digit, 8 bits a pass: a histogram of the keys that share the digits found so far, then the
// digit at which the count from above reaches n.  A last pass in row order writes the rows above that key, and the
// first of those equal to it, behind one another (prefix sums over the workgroup).
// copy_kernel: 16 bytes a thread and step, rows of K and V through both page tables.  Bound: HBM, 4D bytes
// read and 4D written a kept row.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "tfgfa.h"
#include "tfgfa_layout.h"
#include "tfgfa_serving.h"

namespace tfgfa_evict {

using tfgfa::apart;
using tfgfa::Pages;
using tfgfa::pages_ok;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxD = 128;
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

struct Args {
  const int* table;
  const int* lens;
  const float* weights;
  const int* new_table;
  int* kept;
  float* out;
  long long table_stride, new_stride, wb, wh, ob, oh;
  int Hkv, P, page, n_max, budget, recent;
};

// Order of the weight of row j < L as an unsigned number.
__device__ __forceinline__ uint32_t rank_key(float w, bool keep) {
  const uint32_t x = __float_as_uint(w + 0.f);  // -0 as 0
  const uint32_t y = x >> 31 ? ~x : x | 0x80000000u;
  return keep ? 0xFFFFFFFFu : w != w ? 0u : y;
}

// Sum of x over the workgroup's threads before this one; *all: over all of them.
__device__ __forceinline__ int block_before(int x, int* sh, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = y;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? sh[w] : 0;
    sum += sh[w];
  }
  *all = sum;
  return before + y - x;
}

__global__ __launch_bounds__(kThreads) void select_kernel(const Args a) {
  __shared__ int hist[256];
  __shared__ int sh[kWaves];
  __shared__ int sh_digit, sh_above, sh_bad;
  const int tid = threadIdx.x, kv = blockIdx.x, b = blockIdx.y;
  const float* const w = a.weights + b * a.wb + kv * a.wh;
  int* const kept = a.kept + ((long long)b * a.Hkv + kv) * a.budget;
  float* const out = a.out + b * a.ob + kv * a.oh;
  int L = a.lens[b];
  bool bad = L < 0 || L > a.n_max;
  if (bad) L = 0;
  const int n = min(L, a.budget);
  if (tid == 0) sh_bad = 0;
  __syncthreads();
  for (int c = tid; c < (L + a.page - 1) / a.page; c += kThreads)
    bad |= (uint32_t)a.table[b * a.table_stride + c] >= (uint32_t)a.P;
  for (int c = tid; c < (n + a.page - 1) / a.page; c += kThreads)
    bad |= (uint32_t)a.new_table[b * a.new_stride + c] >= (uint32_t)a.P;
  if (bad) sh_bad = 1;
  __syncthreads();
  if (sh_bad) {
    for (int i = tid; i < a.budget; i += kThreads) {
      kept[i] = -1;
      out[i] = __uint_as_float(0x7FC00000u);
    }
    return;
  }
  // The n-th largest key: its digits, and how many of the keys equal to it are wanted.
  uint32_t key = 0;
  int want = n;
  const int old = L - min(L, a.recent);
  if (L > a.budget) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int j = tid; j < L; j += kThreads) {
        const uint32_t x = rank_key(w[j], j >= old);
        if (shift == 24 || (x >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[(x >> shift) & 255], 1);
      }
      __syncthreads();
      int all;
      const int mine = tid < 256 ? hist[255 - tid] : 0;  // from the highest digit down
      const int above = block_before(mine, sh, &all);
      if (tid < 256 && above < want && above + mine >= want) {
        sh_digit = 255 - tid;
        sh_above = above;
      }
      __syncthreads();
      key |= (uint32_t)sh_digit << shift;
      want -= sh_above;
    }
  }
  // In row order: the rows above the key, and the first `want` of those equal to it.
  int done = 0, ties = 0;
  for (int j0 = 0; j0 < L; j0 += kThreads) {
    const int j = j0 + tid;
    const float x = j < L ? w[j] : 0.f;
    bool take = j < L;
    int all;
    if (L > a.budget) {
      const uint32_t y = rank_key(x, j >= old);
      const bool tie = j < L && y == key;
      const int t = block_before(tie ? 1 : 0, sh, &all);
      take = j < L && (y > key || (tie && ties + t < want));
      ties += all;
    }
    const int at = done + block_before(take ? 1 : 0, sh, &all);
    done += all;
    // Every row of this step has been read (the barriers above), and rows move down only: `out` may be `w`.
    if (take) {
      kept[at] = j;
      out[at] = x;
    }
  }
  __syncthreads();
  for (int i = n + tid; i < a.budget; i += kThreads) {
    kept[i] = -1;
    out[i] = 0.f;
  }
}

__global__ __launch_bounds__(256) void copy_kernel(char* k, char* v, Pages ks, Pages vs,
                                                   const int* __restrict__ table, long long table_stride,
                                                   const int* __restrict__ new_table, long long new_stride,
                                                   const int* __restrict__ kept, int Hkv, int page, int budget,
                                                   int pieces) {
  const int kv = blockIdx.y, b = blockIdx.z;
  const int* const rows = kept + ((long long)b * Hkv + kv) * budget;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(x / pieces), c = (int)(x - (long long)i * pieces);
  if (i >= budget) return;
  const int j = rows[i];
  if (j < 0) return;
  const long long from = table[b * table_stride + j / page], to = new_table[b * new_stride + i / page];
  const int fo = j % page, ti = i % page;
  const u32x4 kx = *reinterpret_cast<const u32x4*>(k + from * ks.p + kv * ks.h + fo * ks.n + 16 * c);
  const u32x4 vx = *reinterpret_cast<const u32x4*>(v + from * vs.p + kv * vs.h + fo * vs.n + 16 * c);
  *reinterpret_cast<u32x4*>(k + to * ks.p + kv * ks.h + ti * ks.n + 16 * c) = kx;
  *reinterpret_cast<u32x4*>(v + to * vs.p + kv * vs.h + ti * vs.n + 16 * c) = vx;
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
  const long long grid = ((long long)budget * (D / 8) + 255) / 256;
  if (n_max > INT32_MAX - kThreads || (long long)M_new * page > INT32_MAX || budget > INT32_MAX - kThreads ||
      B > 65535 || H_kv > 65535 || grid > INT32_MAX / 256)
    return TFGFA_ERR_TOO_LARGE;
  if (!k_strides || !v_strides || !weights_strides || !weights_out_strides) return TFGFA_ERR_NULL_POINTER;
  Pages ks, vs;
  if (!pages_ok(k_strides, P, H_kv, page, D, &ks) || !pages_ok(v_strides, P, H_kv, page, D, &vs))
    return TFGFA_ERR_STRIDE;
  if (B > 1 && (table_stride < 0 || new_table_stride < M_new)) return TFGFA_ERR_STRIDE;
  Args a = {};
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
  a.table = page_table, a.lens = cache_seqlens, a.weights = key_weights, a.new_table = new_page_table;
  a.kept = kept, a.out = weights_out;
  a.table_stride = B > 1 ? table_stride : 0, a.new_stride = B > 1 ? new_table_stride : 0;
  a.Hkv = H_kv, a.P = P, a.page = page, a.n_max = (int)n_max, a.budget = budget, a.recent = recent;
  const hipStream_t stream = (hipStream_t)hip_stream;
  hipLaunchKernelGGL(select_kernel, dim3(H_kv, B), dim3(kThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return -(int)e;
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)grid, H_kv, B), dim3(256), 0, stream, static_cast<char*>(k_pages),
                     static_cast<char*>(v_pages), ks, vs, page_table, a.table_stride, new_page_table, a.new_stride,
                     kept, H_kv, page, budget, D / 8);
  e = hipGetLastError();
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
