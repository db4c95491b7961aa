// tfgfa_logits.hip - penalties for repeated tokens, biases and grammar masks on logits, MI355X (gfx950).
//
// Bound: HBM, the logits read and written once.  A workgroup owns kChunk tokens of one row: it counts the
// row's history into LDS (only its own tokens; integer adds, so their order is no matter), then passes over its
// logits once.  The history is read by every workgroup of the row (from L2), which costs less than a counting
// kernel before this one.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "tfgfa.h"
#include "tfgfa_serving.h"

namespace tfgfa_logits {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;

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

template <class E>
__global__ __launch_bounds__(kThreads) void penalize_kernel(const Args a) {
  __shared__ int count[kChunk];
  const int tid = threadIdx.x, b = blockIdx.y, v0 = blockIdx.x * kChunk;
  for (int i = tid; i < kChunk; i += kThreads) count[i] = 0;
  __syncthreads();
  int T = a.T;
  if (a.lengths) T = max(0, min(T, a.lengths[b]));
  for (int t = tid; t < T; t += kThreads) {
    const long long v = (a.token_bytes == 8 ? static_cast<const long long*>(a.tokens)[b * a.ts + t]
                                            : (long long)static_cast<const int*>(a.tokens)[b * a.ts + t]) -
                        v0;
    if (v >= 0 && v < kChunk) atomicAdd(&count[(int)v], 1);
  }
  __syncthreads();
  const float rep = a.reps ? a.reps[b] : a.rep, pres = a.press ? a.press[b] : a.pres,
              freq = a.freqs ? a.freqs[b] : a.freq;
  const E* const x = static_cast<const E*>(a.x) + b * a.xs;
  E* const y = static_cast<E*>(a.y) + b * a.ys;
  for (int i = tid; i < kChunk; i += kThreads) {
    const int v = v0 + i;
    if (v >= a.V) break;
    float z = (float)x[v];
    const int n = count[i];
    if (n > 0) z = (z > 0.f ? z / rep : z * rep) - freq * (float)n - pres;
    if (a.bias) z += a.bias[b * a.bs + v];
    if (a.allowed && !((a.allowed[b * a.as + (v >> 5)] >> (v & 31)) & 1u)) z = -INFINITY;
    y[v] = (E)z;
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
  if (B > 65535 || V > INT32_MAX - kChunk || T > INT32_MAX - kThreads) return TFGFA_ERR_TOO_LARGE;
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
  const dim3 grid((V + kChunk - 1) / kChunk, B);
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (kind == TFSERVE_LOGITS_F32)
    hipLaunchKernelGGL((penalize_kernel<float>), grid, dim3(kThreads), 0, stream, a);
  else if (kind == TFSERVE_LOGITS_BF16)
    hipLaunchKernelGGL((penalize_kernel<__bf16>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((penalize_kernel<_Float16>), grid, dim3(kThreads), 0, stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TFGFA_OK : -(int)e;
}
