// tfgfa_weights.hip - the attention weight that each key receives from given queries, MI355X (gfx950):
//     c_j = sum_h sum_i [j <= first + i] e^(scale q_hi . k_j - lse_hi)
// over the query heads h of a key-value head, with the log-sum-exp of the attention that ran before.
//
// Bound: the exponentials.  A pair of query and key costs 2D flops on the matrix units (64 cycles a 32x32
// tile and 32 dims) and one v_exp_f32, one v_fma and one v_add on the VALU, the first at a quarter of the rate:
// about 384 cycles a tile against 128 at D = 64.
//
// S^T[key][query] = K Q^T as v_mfma_f32_32x32x16 tiles: lane l holds 16 keys of query l % 32, so that the
// query's lse is one register, the sums over queries stay in 16 registers of each lane, and lanes are
// added once at the end.  A workgroup owns 32 keys of one key-value head, whose K rows stay in registers; its
// waves take the (query head, 32 queries) tiles in turn, and their sums are added in wave order.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "tfgfa.h"
#include "tfgfa_layout.h"
#include "tfgfa_serving.h"

namespace tfgfa_weights {

using tfgfa::apart;
using tfgfa::Rows;
using tfgfa::rows_ok;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxD = 128;
constexpr int kTile = 32;
constexpr int kWaves = 4;

template <class T>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma<__bf16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma<_Float16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}

struct Args {
  const void* q;
  const void* k;
  const float* lse;
  float* out;
  Rows qs, ks;
  long long lb, lh, ob, oh;
  long long first;
  float scale_log2;
  int G, Nq, Nk, D, causal;
};

// kP: pieces of 16 dims, D <= 16 kP; a lane holds dims 16p + 8 (l / 32) .. + 7 of row l % 32.
template <class T, int kP>
__global__ __launch_bounds__(64 * kWaves) void weights_kernel(const Args a) {
  __shared__ float sums[kWaves][kTile];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, i = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv = blockIdx.y, b = blockIdx.z, j0 = blockIdx.x * kTile;
  u32x4 kf[kP];
  const T* const kr = static_cast<const T*>(a.k) + b * a.ks.b + kv * a.ks.h + (long long)(j0 + i) * a.ks.n + 8 * half;
#pragma unroll
  for (int p = 0; p < kP; ++p)
    kf[p] = j0 + i < a.Nk && 16 * p + 8 * half < a.D ? *reinterpret_cast<const u32x4*>(kr + 16 * p)
                                                     : u32x4{0, 0, 0, 0};
  // First tile of queries that see a key of this workgroup.
  const int tiles = (a.Nq + kTile - 1) / kTile;
  int t0 = 0;
  if (a.causal && j0 > a.first) t0 = (int)min((long long)tiles, (j0 - a.first) / kTile);
  const int per = tiles - t0;
  float sum[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) sum[r] = 0.f;
  for (int w = wave; w < per * a.G; w += kWaves) {
    const int g = w / per, t = t0 + (w - g * per), h = kv * a.G + g, q0 = t * kTile;
    const bool in = q0 + i < a.Nq;
    const T* const qr = static_cast<const T*>(a.q) + b * a.qs.b + h * a.qs.h + (long long)(q0 + i) * a.qs.n + 8 * half;
    u32x4 qf[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p)
      qf[p] = in && 16 * p + 8 * half < a.D ? *reinterpret_cast<const u32x4*>(qr + 16 * p) : u32x4{0, 0, 0, 0};
    // Keys of the tile that this lane's query sees: up to `last`.  A row past the last, and one with nothing to
    // see (lse -inf, or past the range in the log2 domain), sees none.
    float z = in ? a.lse[b * a.lb + h * a.lh + q0 + i] * kLog2e : INFINITY;
    const bool live = z != INFINITY && z != -INFINITY;
    z = live ? z : 0.f;
    int last = kTile - 1;
    if (a.causal) last = (int)max(-1LL, min((long long)last, a.first + q0 + i - j0));
    if (!live) last = -1;
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int p = 0; p < kP; ++p) s = mfma<T>(kf[p], qf[p], s);
    // Register r: key 8 (r / 4) + 4 half + r % 4 of the tile, query i.
    const bool edge = __builtin_amdgcn_ballot_w64(last < kTile - 1) != 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, -z));
      if (edge) p = 8 * (r / 4) + 4 * half + r % 4 <= last ? p : 0.f;
      sum[r] += p;
    }
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) sum[r] += __shfl_xor(sum[r], o);
    if (i == 0) sums[wave][8 * (r / 4) + 4 * half + r % 4] = sum[r];
  }
  __syncthreads();
  if (tid < kTile && j0 + tid < a.Nk) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x += sums[w][tid];
    a.out[b * a.ob + kv * a.oh + j0 + tid] = x;
  }
}

}  // namespace tfgfa_weights

extern "C" int tfserve_key_weights(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                   const float* lse, const int64_t* lse_strides, float* out,
                                   const int64_t* out_strides, int B, int H, int H_kv, int N_q, int N_k, int D,
                                   int dtype, float softmax_scale, int causal, int64_t first_query,
                                   void* hip_stream) {
  using namespace tfgfa_weights;
  if (dtype != TFGFA_DTYPE_BF16 && dtype != TFGFA_DTYPE_F16) return TFGFA_ERR_DTYPE;
  if (B < 0 || H < 0 || H_kv < 0 || N_q < 0 || N_k < 0 || first_query < 0) return TFGFA_ERR_BAD_SHAPE;
  if (H_kv == 0 ? H != 0 : (H == 0 || H % H_kv != 0)) return TFGFA_ERR_BAD_SHAPE;
  if (D < 8 || D > kMaxD || (D & 7)) return TFGFA_ERR_HEAD_DIM;
  if (!(softmax_scale > 0.f) || !isfinite(softmax_scale)) return TFGFA_ERR_SCALE;
  if (causal != 0 && causal != 1) return TFGFA_ERR_CAUSAL_FLAG;
  if (B == 0 || H == 0 || N_k == 0) return TFGFA_OK;
  if (B > 65535 || H_kv > 65535 || N_q > INT32_MAX - kTile || N_k > INT32_MAX - kTile ||
      first_query > INT64_MAX / 2 || (long long)(N_q / kTile + 1) * (H / H_kv) > INT32_MAX - kWaves)
    return TFGFA_ERR_TOO_LARGE;
  if (!q_strides || !k_strides || !lse_strides || !out_strides) return TFGFA_ERR_NULL_POINTER;
  Args a = {};
  if (!rows_ok(q_strides, B, H, N_q, D, &a.qs) || !rows_ok(k_strides, B, H_kv, N_k, D, &a.ks))
    return TFGFA_ERR_STRIDE;
  if (!k || !out || (N_q > 0 && (!q || !lse))) return TFGFA_ERR_NULL_POINTER;
  if (((uintptr_t)q | (uintptr_t)k) & 15u) return TFGFA_ERR_ALIGNMENT;
  if (((uintptr_t)lse | (uintptr_t)out) & 3u) return TFGFA_ERR_ALIGNMENT;
  a.lb = B > 1 ? lse_strides[0] : 0, a.lh = H > 1 ? lse_strides[1] : 0;
  a.ob = B > 1 ? out_strides[0] : 0, a.oh = H_kv > 1 ? out_strides[1] : 0;
  if (a.lb < 0 || a.lh < 0 || !apart(a.ob, B, a.oh, H_kv, N_k))
    return TFGFA_ERR_STRIDE;
  a.q = q, a.k = k, a.lse = lse, a.out = out;
  a.first = first_query;
  a.scale_log2 = softmax_scale * kLog2e;
  a.G = H / H_kv, a.Nq = N_q, a.Nk = N_k, a.D = D, a.causal = causal;
  const dim3 grid((N_k + kTile - 1) / kTile, H_kv, B);
  const hipStream_t stream = (hipStream_t)hip_stream;
#define TFGFA_WEIGHTS(T)                                                                            \
  do {                                                                                              \
    if (D <= 64)                                                                                    \
      hipLaunchKernelGGL((weights_kernel<T, 4>), grid, dim3(64 * kWaves), 0, stream, a);            \
    else                                                                                            \
      hipLaunchKernelGGL((weights_kernel<T, 8>), grid, dim3(64 * kWaves), 0, stream, a);            \
  } while (0)
  if (dtype == TFGFA_DTYPE_BF16)
    TFGFA_WEIGHTS(__bf16);
  else
    TFGFA_WEIGHTS(_Float16);
#undef TFGFA_WEIGHTS
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
