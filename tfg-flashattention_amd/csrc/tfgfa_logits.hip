// tfgfa_logits.hip - penalties for repeated tokens, biases and grammar masks on logits, MI355X (gfx950).
//
// Bound: HBM, the logits read and written once.  A workgroup owns a chunk of one row, whose logits, biases and mask
// words it asks for first; while they come it counts the row's history into LDS (its own tokens only; integer adds,
// so their order is no matter), which every workgroup of the row reads from L2.  Rows of odd lengths begin at any
// element: a lane takes four neighbouring logits as one load of the elements' own alignment.
// Measured: 128 rows of 50257 float32 logits with biases, masks and 1024 tokens each, 53.5 MB in 12.8 us (4.2 TB/s;
// 11.7 where the Infinity Cache holds them); one row 3.0 us.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "tfgfa.h"
#include "tfgfa_serving.h"

namespace tfgfa_logits {

constexpr int kThreads = 256;
constexpr int kEach = 4;              // neighbouring logits of a lane
constexpr int kMaxSteps = 4, kFewSteps = 1;  // of kThreads * kEach logits in a chunk
constexpr int kTokens = 4;            // tokens of the history that a lane loads at once

struct Args {
  const void* x;
  void* y;
  const void* tokens;
  const int* lengths;
  const float* reps;
  const float* press;
  const float* freqs;
  const float* bias;
  const uint32_t* allowed;
  long long xs, ys, ts, bs, as;
  float rep, pres, freq;
  int token_bytes, V, T;
};

// kEach neighbouring values of type E at any element.
template <class E>
struct Pack {
  typedef E v __attribute__((ext_vector_type(kEach)));
  typedef v __attribute__((aligned(sizeof(E)))) any;
};

// kSteps: of kThreads * kEach logits in a workgroup's chunk.
template <class E, int kSteps>
__global__ __launch_bounds__(kThreads) void penalize_kernel(const Args a) {
  constexpr int kChunk = kThreads * kEach * kSteps;
  __shared__ int count[kChunk];
  const int tid = threadIdx.x, b = blockIdx.y, v0 = blockIdx.x * kChunk;
  const E* const x = static_cast<const E*>(a.x) + b * a.xs;
  E* const y = static_cast<E*>(a.y) + b * a.ys;
  const float* const bias = a.bias ? a.bias + b * a.bs : nullptr;
  const uint32_t* const allowed = a.allowed ? a.allowed + b * a.as : nullptr;
  typename Pack<E>::v z[kSteps];
  typename Pack<float>::v w[kSteps];
  uint32_t bits[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int v = v0 + (s * kThreads + tid) * kEach;  // (a multiple of 4: its four bits are in one word)
    if (v + kEach <= a.V) {
      z[s] = *reinterpret_cast<const typename Pack<E>::any*>(x + v);
      if (bias) w[s] = *reinterpret_cast<const typename Pack<float>::any*>(bias + v);
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        z[s][e] = v + e < a.V ? x[v + e] : (E)0.f;
        if (bias) w[s][e] = v + e < a.V ? bias[v + e] : 0.f;
      }
    }
    bits[s] = allowed && v < a.V ? allowed[v >> 5] >> (v & 31) : 0xFu;
  }
  int T = a.T;
  if (a.lengths) T = max(0, min(T, a.lengths[b]));
  const float rep = a.reps ? a.reps[b] : a.rep, pres = a.press ? a.press[b] : a.pres,
              freq = a.freqs ? a.freqs[b] : a.freq;
#pragma unroll
  for (int s = 0; s < kSteps * kEach; ++s) count[s * kThreads + tid] = 0;
  __syncthreads();
  for (int t0 = 0; t0 < T; t0 += kThreads * kTokens) {
    long long id[kTokens];
#pragma unroll
    for (int c = 0; c < kTokens; ++c) {
      const int t = t0 + c * kThreads + tid;
      id[c] = -1;
      if (t < T)
        id[c] = a.token_bytes == 8 ? static_cast<const long long*>(a.tokens)[b * a.ts + t]
                                   : (long long)static_cast<const int*>(a.tokens)[b * a.ts + t];
    }
#pragma unroll
    for (int c = 0; c < kTokens; ++c)
      if (id[c] >= v0 && id[c] < v0 + kChunk) atomicAdd(&count[(int)(id[c] - v0)], 1);
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int at = (s * kThreads + tid) * kEach, v = v0 + at;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const i32x4 n = *reinterpret_cast<const i32x4*>(&count[at]);
    typename Pack<E>::v out;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      float f = (float)z[s][e];
      if (n[e] > 0) f = (f > 0.f ? f / rep : f * rep) - freq * (float)n[e] - pres;
      if (bias) f += w[s][e];
      out[e] = (E)((bits[s] >> e) & 1u ? f : -INFINITY);
    }
    if (v + kEach <= a.V) {
      *reinterpret_cast<typename Pack<E>::any*>(y + v) = out;
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (v + e < a.V) y[v + e] = out[e];
    }
  }
}

}  // namespace tfgfa_logits

extern "C" int tfserve_penalize(const void* logits, int64_t logits_stride, void* out, int64_t out_stride, int kind,
                                const void* tokens, int token_bytes, int64_t tokens_stride, const int* lengths,
                                const float* repetitions, float repetition, const float* presences, float presence,
                                const float* frequencies, float frequency, const float* bias, int64_t bias_stride,
                                const int* allowed, int64_t allowed_stride, int B, int V, int T, void* hip_stream) {
  using namespace tfgfa_logits;
  if (kind != TFSERVE_LOGITS_BF16 && kind != TFSERVE_LOGITS_F16 && kind != TFSERVE_LOGITS_F32)
    return TFGFA_ERR_DTYPE;
  if (token_bytes != 4 && token_bytes != 8) return TFGFA_ERR_DTYPE;
  if (B < 0 || V < 0 || T < 0) return TFGFA_ERR_BAD_SHAPE;
  if (!repetitions && (!(repetition > 0.f) || !isfinite(repetition))) return TFGFA_ERR_SCALE;
  if ((!presences && !isfinite(presence)) || (!frequencies && !isfinite(frequency))) return TFGFA_ERR_SCALE;
  if (B == 0 || V == 0) return TFGFA_OK;
  if (B > 65535 || V > INT32_MAX - kThreads * kEach * kMaxSteps || T > INT32_MAX - kThreads * kTokens) return TFGFA_ERR_TOO_LARGE;
  if (B > 1 && (logits_stride < 0 || out_stride < V || (T > 0 && tokens_stride < 0) || bias_stride < 0 ||
                allowed_stride < 0))
    return TFGFA_ERR_STRIDE;
  if (!logits || !out || (T > 0 && !tokens)) return TFGFA_ERR_NULL_POINTER;
  if (out == logits && B > 1 && logits_stride != out_stride) return TFGFA_ERR_STRIDE;
  const uintptr_t size = kind == TFSERVE_LOGITS_F32 ? 4 : 2;
  if ((((uintptr_t)logits | (uintptr_t)out) & (size - 1)) || ((uintptr_t)tokens & (token_bytes - 1)) ||
      (((uintptr_t)lengths | (uintptr_t)repetitions | (uintptr_t)presences | (uintptr_t)frequencies |
        (uintptr_t)bias | (uintptr_t)allowed) & 3u))
    return TFGFA_ERR_ALIGNMENT;
  Args a = {};
  a.x = logits, a.y = out, a.tokens = tokens, a.lengths = lengths;
  a.reps = repetitions, a.press = presences, a.freqs = frequencies, a.bias = bias;
  a.allowed = reinterpret_cast<const uint32_t*>(allowed);
  if (B > 1) a.xs = logits_stride, a.ys = out_stride, a.ts = tokens_stride, a.bs = bias_stride, a.as = allowed_stride;
  a.rep = repetition, a.pres = presence, a.freq = frequency;
  a.token_bytes = token_bytes, a.V = V, a.T = T;
  int cu = 0;
  const int st = tfgfa_device_info(&cu, nullptr, nullptr, 0);
  if (st != TFGFA_OK) return st;
  // Long chunks where they make workgroups enough, four a CU: each reads its row's history.  (1 row of 50257: 3.5 us
  // with short ones, 4.7 with long ones; 128 rows 12.3 both.)
  const int steps = (long long)B * (V / (kThreads * kEach * kMaxSteps)) >= 4LL * cu ? kMaxSteps : kFewSteps;
  const dim3 grid((V + kThreads * kEach * steps - 1) / (kThreads * kEach * steps), B);
  const hipStream_t stream = (hipStream_t)hip_stream;
#define TFGFA_PENALIZE(E)                                                                            \
  do {                                                                                               \
    if (steps == kMaxSteps)                                                                          \
      hipLaunchKernelGGL((penalize_kernel<E, kMaxSteps>), grid, dim3(kThreads), 0, stream, a);       \
    else                                                                                             \
      hipLaunchKernelGGL((penalize_kernel<E, kFewSteps>), grid, dim3(kThreads), 0, stream, a);       \
  } while (0)
  if (kind == TFSERVE_LOGITS_F32)
    TFGFA_PENALIZE(float);
  else if (kind == TFSERVE_LOGITS_BF16)
    TFGFA_PENALIZE(__bf16);
  else
    TFGFA_PENALIZE(_Float16);
#undef TFGFA_PENALIZE
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
